// Linear layer in 8-bit floating point (e4m3) with a scale for each block of 128:
//   y[m, n] = sum_b s[m, b] t[n / 128, b] (sum_{k in block b} q[m, k] w[n, k]) (+ bias[n]),
// w the weights in e4m3 with one fp32 scale t per 128 x 128 block, q the activations, quantized on the way in with one
// scale s per token and 128 values: with a = max(max |x|, 2^-100), q = e4m3(x (448 / a)) rounded to nearest even and
// s = a / 448, in fp32. Products of e4m3 values are exact in fp32; a block's sum comes from the tensor core, the sum over
// blocks is held in fp32 registers with one multiply-add a block, and the result is rounded once.
#include <atomic>
#include <climits>

#include "lb_launch.h"
#include "lb_tc.cuh"
#include "lb_types.cuh"

namespace lb {

// status word of this file's kernels (a bounded wait that gave up)
__device__ int g_f8_status;

namespace {

constexpr int kBlock = 128;               // values of a scale
constexpr float kMost = 448.f;            // largest e4m3 value
constexpr float kLeast = 0x1p-100f;       // blocks whose maximum is below count as if it were this

__device__ __forceinline__ float lds_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
// two fp32 values in one 64-bit register pair
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// ------------------------------------------------------------------------------------------------------- quantize
// a block's scale and its inverse; a maximum that is not finite makes the scale so, and with it what the row gives
struct BlockScale {
  float up, s;
};
__device__ __forceinline__ BlockScale block_scale(uint32_t amax_bits) {
  const float a = fmaxf(__uint_as_float(amax_bits), kLeast);   // (fmaxf drops a NaN: it is put back below)
  BlockScale v;
  v.up = kMost / a;
  v.s = amax_bits > 0x7F800000u ? __uint_as_float(amax_bits) : a / kMost;
  return v;
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | (uint32_t)hi << 16;
}
__device__ __forceinline__ uint2 e4m3x8(const float (&f)[8], float up) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(f[i], up);
  return make_uint2(e4m3x4(v[0], v[1], v[2], v[3]), e4m3x4(v[4], v[5], v[6], v[7]));
}

// eight values of a row from p on, zeros behind the n that are left; through L2 only (the row may have been written while
// this kernel was already resident)
template <typename T>
__device__ __forceinline__ uint4 load8(const T* p, int n, bool aligned) {
  if (n >= 8 && aligned) return ldg_cg_u128(p);
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = i < n ? (uint32_t)ldg_cg_u16(p + i) : 0u;
  return make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
}
template <typename T>
__device__ __forceinline__ void floats8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = Elem<T>::unpack(w[i]);
    f[2 * i] = a.x;
    f[2 * i + 1] = a.y;
  }
}
// max |x| of eight values on the bits without the sign, which order like the magnitudes with NaN above all
__device__ __forceinline__ uint32_t amax8(const float (&f)[8]) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(f[i]) & 0x7FFFFFFFu);
  return a;
}

// max |x| of eight 16-bit values as fp32 bits: the values' bits without the sign order like the magnitudes, NaN above all
template <typename T>
__device__ __forceinline__ uint32_t amax_packed(const uint4& v) {
  const uint32_t m = 0x7FFF7FFFu;
  const uint32_t a = __vmaxu2(__vmaxu2(v.x & m, v.y & m), __vmaxu2(v.z & m, v.w & m));
  return __float_as_uint(Elem<T>::unpack(max(a & 0xFFFFu, a >> 16)).x);
}

// Tokens: 16 lanes take a block of 128 values, a warp two tokens, a CTA 16 tokens x QB blocks, all of whose loads are
// under way at once. The scales go to [block][token], as the product reads them, 16 tokens a run. Bound by memory: 8192 tokens
// of 18944 values 92 us, 5.0 TB/s.
enum Release { kAtEnd, kAfterWait, kAtEntry };   // when the quantization lets the next kernel start

template <typename T, int QB>
__global__ void __launch_bounds__(256)
    f8_tokens_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, int ldq, float* __restrict__ s, int lds,
                     int M, int K, int release) {
  if (release == kAtEntry) pdl_launch_dependents();
  pdl_wait();
  if (release == kAfterWait) pdl_launch_dependents();
  const int g = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int m = blockIdx.y * 16 + g, b0 = blockIdx.x * QB;
  const bool aligned = ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(ldx * sizeof(T))) & 15u) == 0;
  const T* row = x + (int64_t)min(m, M - 1) * ldx;
  uint4 v[QB];
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int k = (b0 + i) * kBlock + 8 * lane;
    v[i] = k < K ? load8(row + k, K - k, aligned) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int b = b0 + i, k = b * kBlock + 8 * lane;
    float f[8];
    floats8<T>(v[i], f);
    uint32_t a = amax_packed<T>(v[i]);
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, d));
    const BlockScale sc = block_scale(a);
    if (m < M && b * kBlock < K) {
      if (k < ldq) *reinterpret_cast<uint2*>(q + (int64_t)m * ldq + k) = e4m3x8(f, sc.up);
      if (lane == 0) s[(int64_t)b * lds + m] = sc.s;
    }
  }
}

// Weights: a CTA a 128 x 128 block, 16 lanes a row.
template <typename T>
__device__ __forceinline__ void load_floats(const T* p, int n, float (&f)[8]) {
  floats8<T>(load8(p, n, (reinterpret_cast<uintptr_t>(p) & 15u) == 0), f);
}
template <>
__device__ __forceinline__ void load_floats<float>(const float* p, int n, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = i < n ? __uint_as_float(ldg_cg_u32(reinterpret_cast<const uint32_t*>(p + i))) : 0.f;
}

template <typename T>
__global__ void __launch_bounds__(256)
    f8_weight_kernel(const T* __restrict__ w, int64_t ldw, uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ t, int N,
                     int K) {
  __shared__ uint32_t most;
  if (threadIdx.x == 0) most = 0u;
  __syncthreads();
  pdl_wait();
  const int k = blockIdx.x * kBlock + 8 * (threadIdx.x & 15), n0 = blockIdx.y * kBlock + (threadIdx.x >> 4);
  float f[8][8];
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = n0 + 16 * i;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
    if (n < N && k < K) load_floats<T>(w + (int64_t)n * ldw + k, K - k, f[i]);
    a = max(a, amax8(f[i]));
  }
  a = __reduce_max_sync(0xffffffffu, a);
  if ((threadIdx.x & 31) == 0) atomicMax(&most, a);
  __syncthreads();
  const BlockScale sc = block_scale(most);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = n0 + 16 * i;
    if (n < N && k < ldq) *reinterpret_cast<uint2*>(q + (int64_t)n * ldq + k) = e4m3x8(f[i], sc.up);
  }
  if (threadIdx.x == 0) t[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = sc.s;
}

// ------------------------------------------------------------------------------------------------------- the product, few tokens
// tcgen05.mma kind::f8f6f4 with the channels as the A side (128 a CTA, which is a row of the weights' blocks) and a tile of
// bn tokens as the N side. A stage of the ring is 128 bytes of K, so one block of the scales: each stage's four MMAs start a
// new accumulator, and 16 epilogue warps add it, times s t, to the sums that they hold in registers (a lane a channel, a
// column a token) while the next stages' MMAs run into the other accumulators. The scale of a column is the same for all
// lanes: each warp puts its columns' s t into shared memory, from where four come in one broadcast load; two columns take
// one fp32-pair multiply-add.
// CTAs are persistent over tiles, tokens innermost. Few tiles and long K: a cluster of S CTAs splits K, each parks
// its fp32 partial tile in its idle ring, and all sum their share of the outputs through distributed shared memory in rank order.
constexpr int kChunk = 128;               // bytes of K per stage
constexpr int kWBytes = 128 * kChunk;
constexpr int kEpiWarps = 16;
constexpr int kMmaThreads = (2 + kEpiWarps) * 32;   // loader, MMA, epilogue warps
constexpr int kMaxStages = 8;
constexpr int kMaxAcc = 8;
constexpr int kMaxSplits = 8;             // portable cluster size
constexpr int kSmem = 227 * 1024;
constexpr int kBarrierBytes = (2 * kMaxStages + 2 * kMaxAcc) * 8 + 16 + kEpiWarps * (2 * 64 * 4 + 1024);   // + scales, + staging

struct F8Gemm {
  const float* s;       // token scales [blocks][lds]
  const float* t;       // weight scales [rows of blocks][blocks]
  const void* bias;
  void* y;
  int M, N, chunks, lds;
  int bn, tiles_m, tiles, splits, stages;
  int acc, acc_stride;  // accumulators (a power of two) and the columns between them
  int park;             // byte offset behind the ring: barriers, scales, staging
  bool vec;             // output rows take 16-byte stores
};

// This CTA's share of a cluster's outputs: the fp32 partial tiles [token][128 channels] at the same offset of every CTA's
// shared memory, summed in rank order
template <typename T>
__device__ __forceinline__ void sum_partials(uint32_t red, const T* bias, T* y, int n0, int N, int rows, int rank, int S) {
  const int r4 = (threadIdx.x & 31) * 4;
  float bn[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) bn[j] = bias && n0 + r4 + j < N ? Elem<T>::to_float(bias[n0 + r4 + j]) : 0.f;
  cluster_sync_all();
  const int warps = blockDim.x >> 5;
  const bool vec = n0 + r4 + 4 <= N && N % 4 == 0 && (reinterpret_cast<uintptr_t>(y) & 7u) == 0;
  for (int m = rank * warps + (threadIdx.x >> 5); m < rows; m += S * warps) {
    const uint32_t off = red + (uint32_t)(m * 128 + r4) * 4u;
    float4 f[kMaxSplits];
#pragma unroll
    for (int q = 0; q < kMaxSplits; ++q)
      if (q < S) f[q] = ld_dsmem_f4(mapa_shared(off, (uint32_t)q));
    float o[4] = {f[0].x, f[0].y, f[0].z, f[0].w};
#pragma unroll
    for (int q = 1; q < kMaxSplits; ++q)
      if (q < S) o[0] += f[q].x, o[1] += f[q].y, o[2] += f[q].z, o[3] += f[q].w;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += bn[j];
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

template <typename T, int NB>   // NB: 16-column blocks of a tile a warp holds, bn <= 64 NB
__global__ void __launch_bounds__(kMmaThreads, 1)
    f8_cols_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap qmap, const F8Gemm p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + p.park);
  uint64_t* empty = full + kMaxStages;
  uint64_t* acc_full = empty + kMaxStages;
  uint64_t* acc_empty = acc_full + kMaxAcc;
  uint32_t* slot = reinterpret_cast<uint32_t*>(acc_empty + kMaxAcc);
  float* scales = reinterpret_cast<float*>(slot + 4);            // [epilogue warps][2][64]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stage_bytes = kWBytes + p.bn * kChunk, S = p.splits, St = p.stages, A = p.acc;
  const int rank = S > 1 ? (int)cluster_rank() : 0;
  const int first = blockIdx.x / S, step = gridDim.x / S;
  const int c0 = p.chunks * rank / S, nc = p.chunks * (rank + 1) / S - c0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < St; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < A; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kEpiWarps);
    }
    mbar_fence_init();
  }
  const uint32_t columns = (uint32_t)(A * p.acc_stride);
  if (warp == 1) tc::alloc(slot, columns);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *slot;
  pdl_launch_dependents();

  if (warp == 0) {
    if (tc::elect_one()) {
      tma_prefetch_map(&wmap);
      tma_prefetch_map(&qmap);
      struct Place {
        int tile, c, m0, n0;
      };
      auto at = [&](int tile) {
        const int n = tile / p.tiles_m, m = tile - n * p.tiles_m;
        return Place{tile, 0, m * p.bn, n * 128};
      };
      auto next = [&](Place& q) {
        if (++q.c == nc) q = at(q.tile + step);
      };
      auto weights = [&](const Place& q, int s) {
        mbar_arrive_expect_tx(&full[s], stage_bytes);
        tma_load_2d(ring + s * stage_bytes, &wmap, (c0 + q.c) * kChunk, q.n0, &full[s]);
      };
      auto tokens = [&](const Place& q, int s) {
        tma_load_2d(ring + s * stage_bytes + kWBytes, &qmap, (c0 + q.c) * kChunk, q.m0, &full[s]);
      };
      Place w = at(first), q = w;
      int head = 0;
      for (; head < St && w.tile < p.tiles; ++head, next(w)) weights(w, head);
      pdl_wait();
      for (int s = 0; s < head; ++s, next(q)) tokens(q, s);
      int s = 0, phase = 0;   // the stage to fill next, and the parity of its release
      bool ok = true;
      for (; q.tile < p.tiles; next(q)) {
        ok = wait_bounded(&empty[s], phase, &g_f8_status);
        if (!ok) break;
        weights(q, s);
        tokens(q, s);
        if (++s == St) s = 0, phase ^= 1;
      }
      // no copy in flight past this point: stage s holds the oldest of the last `head` copies, its parity is that of the
      // release before it
      for (int i = 0; i < head; ++i) {
        wait_bounded(&full[s], phase, &g_f8_status);
        if (++s == head) s = 0, phase ^= 1;
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (tc::elect_one()) {
      // fp32 accumulator, e4m3 A and B, both K-major
      const uint32_t idesc = (1u << 4) | ((uint32_t)(p.bn >> 3) << 17) | ((128u >> 4) << 24);
      const uint64_t desc0 = tc::desc_sw128(smem_addr(ring), 16, 1024);   // the address field counts 16 bytes
      const uint32_t stage_step = (uint32_t)stage_bytes >> 4;
      int s = 0, phase = 0, a = 0, turn = 0;   // stage, its parity; accumulator, times round their ring
      bool ok = true;
      for (int tile = first; tile < p.tiles && ok; tile += step)
        for (int c = 0; c < nc && ok; ++c) {
          if (turn > 0) ok = wait_bounded(&acc_empty[a], (turn - 1) & 1, &g_f8_status);
          if (ok) ok = wait_bounded(&full[s], phase, &g_f8_status);
          if (!ok) break;
          tc::fence_after();
          const uint64_t ad = desc0 + s * stage_step, bd = ad + (kWBytes >> 4);
          const uint32_t d = tmem + a * p.acc_stride;
#pragma unroll
          for (int k = 0; k < 4; ++k) tc::mma_f8_ss(d, ad + 2 * k, bd + 2 * k, idesc, k > 0);
          tc::commit(&empty[s]);
          tc::commit(&acc_full[a]);
          if (++s == St) s = 0, phase ^= 1;
          if (++a == A) a = 0, ++turn;
        }
      // no MMA in flight past this point
      for (int i = 0; i < A; ++i) {
        const int uses = i < a ? turn + 1 : turn;
        if (uses > 0) wait_bounded(&acc_full[i], (uses - 1) & 1, &g_f8_status);
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, part = (warp - 2) >> 2, row = 32 * quarter + lane;
    const uint32_t tlane = tmem + ((uint32_t)(32 * quarter) << 16) + 16 * part;
    const T* bias = static_cast<const T*>(p.bias);
    T* y = static_cast<T*>(p.y);
    float* scale = scales + (warp - 2) * 128;
    uint16_t* turn = reinterpret_cast<uint16_t*>(scales + kEpiWarps * 128) + (warp - 2) * 512;
    pdl_wait();
    bool ok = true;   // of this lane: one that gave up waits no more, but stays with its warp's collective instructions
    int a = 0, phase = 0;
    const int blocks = (p.bn - 16 * part + 63) / 64;   // of this warp
    for (int tile = first; tile < p.tiles; tile += step) {
      const int m0 = tile % p.tiles_m * p.bn, nt = tile / p.tiles_m, n = nt * 128 + row;
      const bool on = n < p.N;
      // this lane's columns' scales and the tile's, one chunk ahead
      constexpr int kCols = NB > 2 ? 2 : 1;
      const float* sp[kCols];
      bool have[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        const int at = lane + 32 * i, col = 64 * (at >> 4) + 16 * part + (at & 15);
        have[i] = at < 16 * NB && col < p.bn && m0 + col < p.M;
        sp[i] = p.s + (int64_t)c0 * p.lds + m0 + col;
      }
      const float* tp = p.t + (int64_t)nt * p.chunks + c0;
      float sv[kCols], tv;
      auto fetch = [&](int c) {
        tv = c < nc ? __ldcg(tp + c) : 0.f;
#pragma unroll
        for (int i = 0; i < kCols; ++i) sv[i] = c < nc && have[i] ? __ldcg(sp[i] + (int64_t)c * p.lds) : 0.f;
      };
      fetch(0);
      uint64_t sum[NB][8];
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[i][j] = 0;
      for (int c = 0; c < nc; ++c) {
        float* sc = scale + 64 * (c & 1);   // (a lane a chunk ahead writes the other half)
#pragma unroll
        for (int i = 0; i < kCols; ++i)
          if (lane + 32 * i < 16 * NB) sc[lane + 32 * i] = sv[i] * tv;
        fetch(c + 1);
        if (ok) ok = wait_bounded(&acc_full[a], phase, &g_f8_status);
        __syncwarp();
        tc::fence_after();
        const uint32_t acc = tlane + (uint32_t)(a * p.acc_stride);
#pragma unroll
        for (int i = 0; i < NB; ++i)
          if (i < blocks) {
            uint32_t v[16];
            tc::ld16(acc + 64 * i, v);
            const ulonglong2* s2 = reinterpret_cast<const ulonglong2*>(sc + 16 * i);
            ulonglong2 f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = s2[j];
            tc::wait_ld();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              sum[i][2 * j] = fma2(pair(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1])), f[j].x, sum[i][2 * j]);
              sum[i][2 * j + 1] = fma2(pair(__uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3])), f[j].y, sum[i][2 * j + 1]);
            }
          }
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[a]);
        if (++a == A) a = 0, phase ^= 1;
      }
      const float bn = on && bias && S == 1 ? Elem<T>::to_float(bias[n]) : 0.f;
#pragma unroll
      for (int i = 0; i < NB; ++i)
        if (i < blocks) {
          const int j0 = 64 * i + 16 * part;
          if (S == 1) {
            const int left = p.M - m0 - j0;   // tokens
            uint32_t h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 v = unpair(sum[i][j]);
              h[j] = Elem<T>::pack(v.x + bn, v.y + bn);
            }
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
            float* red = reinterpret_cast<float*>(ring);   // [token][128 channels]
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 v = unpair(sum[i][j]);
              red[(j0 + 2 * j) * 128 + row] = v.x;
              red[(j0 + 2 * j + 1) * 128 + row] = v.y;
            }
          }
        }
    }
  }
  __syncwarp();
  if (S > 1) {
    const int n0 = first / p.tiles_m * 128, m0 = first % p.tiles_m * p.bn;
    sum_partials<T>(smem_addr(ring), static_cast<const T*>(p.bias), static_cast<T*>(p.y) + (int64_t)m0 * p.N, n0, p.N,
                    min(p.bn, p.M - m0), rank, S);
  }
  tc::fence_before();
  if (S > 1)
    cluster_sync_all();   // no CTA leaves while another still reads its shared memory
  else
    __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    tc::dealloc(tmem, columns);
  }
}

// ------------------------------------------------------------------------------------------------------- the product, many tokens
// The same with the tokens as the A side: a pair of CTAs (cta_group::2) works on 256 tokens, 128 a CTA, and a tile of bn
// channels, half of them loaded by each. A lane now holds a token, so that its scale is one register: s t of a block
// multiplies all columns, without the loads from shared memory that a scale a column takes. A stage's MMAs go into two
// accumulators of about bn / 2 channels, each with an MMA warp and four epilogue warps a CTA of its own, and there are two of
// each in tensor memory, which then is full: what counts is how long one is away, from its first MMA until its last column has
// been read and the issuing thread knows, which is 1700 clocks. So a barrier is asked ahead of the work before it (a completed
// one costs 200 clocks all the same), accumulators are handed back without a release (one at the cluster's scope waits for
// everything in flight: 1840 us a call where this takes 615), scales come with the stage by tensor copies.
// Bound by that way round, 890 clocks a stage of 256 x 224 x 128 for 480 of MMAs: 8192 x 18944 x 3584 615 to 650 us with the
// quantization, 720 under the power cap after a second of calls, 4096 x 4096 x 3584 82. Without the epilogue's multiply-adds a stage
// takes 700 clocks. Left out: four accumulators of 64 channels (700 us), sixteen epilogue warps (646: five warps a scheduler
// slow the MMA warps down), one MMA warp for both halves (738), tiles of 256 channels where 224 fill the last round (740).
constexpr int kRowsSmem = 2 * 1024;       // a warp's staging: 32 tokens x 32 channels
constexpr int kRowsThreads = 12 * 32;     // two loaders and two MMA warps (a warpgroup), 8 epilogue warps
constexpr int kRowsStages = 6;
constexpr int kRowsBarriers = 256;        // bytes, with tensor memory's address; the scales behind them are tensor copies
constexpr int kRowsBarrierBytes = kRowsBarriers + (kRowsStages + 2) * 512 + 8 * kRowsSmem;
static_assert((2 * kRowsStages + 8) * 8 + 16 <= kRowsBarriers && kRowsStages % 2 == 0, "barriers: the accumulators' aligned to 32 bytes");

// the two accumulators' channels, multiples of 32 as a pair's MMA takes them
__host__ __device__ constexpr int first_half(int bn) { return (bn + 63) / 64 * 32; }

struct F8Rows {
  const float* t;       // weight scales [rows of blocks][blocks]
  const void* bias;
  void* y;
  int M, N, chunks;
  int bn, tiles_m, tiles_n, tiles, stages;   // bn a multiple of 32
  int park;             // byte offset behind the ring: barriers, staging
  bool vec;             // output rows take 16-byte stores
};

// The tile at a place of the order in which they are taken: eight columns of tiles at a time, so that what is worked on at one
// moment is about as many tokens as channels, and the fewest rows of both are read.
constexpr int kTileColumns = 8;
struct TilePlace {
  int m, n;
};
__device__ __forceinline__ TilePlace tile_place(int tile, int tiles_m, int tiles_n) {
  const int group = tile / (kTileColumns * tiles_m), rest = tile - group * kTileColumns * tiles_m;
  const int wide = min(kTileColumns, tiles_n - group * kTileColumns), m = rest / wide;
  return {m, group * kTileColumns + rest - m * wide};
}

struct F8Epilogue {
  uint32_t acc_full, acc_empty, scales, tmem;   // shared-memory addresses, acc_empty the leader's
  uint8_t* staging;
  int rank, first, step, n_off, half;
};

// An epilogue warp's work on its B blocks of 16 channels and 32 tokens of every tile
template <typename T, int B>
__device__ __forceinline__ void rows_epilogue(const F8Rows& p, const F8Epilogue& w) {
  const int lane = threadIdx.x & 31, quarter = (threadIdx.x >> 5) & 3, row = 32 * quarter + lane, rank = w.rank, h = w.half;
  const T* bias = static_cast<const T*>(p.bias);
  T* y = static_cast<T*>(p.y);
  uint8_t* stage = w.staging;
  bool ok = true;   // of the warp, as are the waits' answers: having given up it waits no more, but stays with the collective instructions
  bool ready = false;   // the next accumulator, as asked under the work on this one; all lanes found it so
  // of the accumulator: its barrier, that of its release, its columns, the parity of its uses (the turns are 16 bytes and 256
  // columns apart, both aligned to twice that); and the place of the stage's scale
  uint32_t bar = w.acc_full + 8 * h, empty = w.acc_empty + 8 * h, acc = w.tmem + ((uint32_t)(32 * quarter) << 16) + 128 * h, parity = 0, odd = 0;
  const uint32_t scale0 = w.scales + 4 * row, scale_end = scale0 + 512 * (p.stages + 2);
  uint32_t scale = scale0;
  for (int tile = w.first; tile < p.tiles; tile += w.step) {
    const TilePlace at = tile_place(tile, p.tiles_m, p.tiles_n);
    const int m0 = at.m * 256 + 128 * rank, n0 = at.n * p.bn + w.n_off;
    // up to 128 channels: the blocks from `turn` on belong to the next row of the weights' scales
    const int nb = n0 / kBlock, most = (p.N - 1) / kBlock, turn = ((nb + 1) * kBlock - n0) / 16;
    const float* t0 = p.t + (int64_t)min(nb, most) * p.chunks;
    const float* t1 = p.t + (int64_t)min(nb + 1, most) * p.chunks;
    // the weights' scales of 32 stages at a time, a lane a stage, loaded 32 stages before their use
    float ta = 0.f, tb = 0.f, ta2 = 0.f, tb2 = 0.f;
    auto fetch = [&](int c) {
      if (c + lane < p.chunks) ta2 = __ldcg(t0 + c + lane), tb2 = __ldcg(t1 + c + lane);
    };
    fetch(0);
    float sum[B][16];
#pragma unroll
    for (int i = 0; i < B; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) sum[i][j] = 0.f;
    for (int c = 0; c < p.chunks; ++c) {
      if (c % 32 == 0) {
        ta = ta2, tb = tb2;
        fetch(c + 32);
      }
      float fa, fb;
      if (ok && !ready) ok = wait_warp(bar, parity, &g_f8_status);
      __syncwarp();
      tc::fence_after();
      bar ^= 16;
      parity ^= odd;
      odd ^= 1;
      uint32_t v[16];
#pragma unroll
      for (int i = 0; i < B; ++i) {
        tc::ld16(acc + 16 * i, v);
        if (i == 0) {
          const float sv = lds_f32(scale);   // there, since the MMAs have waited for it
          // The arrival below hands back the scale's place too, where a tensor copy puts that of a later stage: its address hangs on a
          // vote for which every lane has to have its scale (rank >> 1 is 0, which the compiler does not know)
          empty += __ballot_sync(0xffffffffu, __float_as_uint(sv) != 0u) & (uint32_t)rank >> 1;
          ready = __all_sync(0xffffffffu, test_barrier(bar, parity));
          fa = __shfl_sync(0xffffffffu, ta, c & 31) * sv;
          fb = __shfl_sync(0xffffffffu, tb, c & 31) * sv;
        }
        tc::wait_ld();
        const float f = i < turn ? fa : fb;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          // two columns in one instruction, as one block of code: what the compiler is left to pair up it copies first
          asm("{\n\t.reg .b64 a, b, c;\n\t"
              "mov.b64 a, {%2, %3};\n\t"
              "mov.b64 b, {%4, %4};\n\t"
              "mov.b64 c, {%0, %1};\n\t"
              "fma.rn.f32x2 c, a, b, c;\n\t"
              "mov.b64 {%0, %1}, c;\n\t}"
              : "+f"(sum[i][2 * j]), "+f"(sum[i][2 * j + 1])
              : "r"(v[2 * j]), "r"(v[2 * j + 1]), "f"(f));
      }
      tc::fence_before();
      __syncwarp();
      tc::arrive_relaxed(empty, lane == 0);
      empty ^= 16;
      acc ^= 256;
      scale += 512;
      if (scale == scale_end) scale = scale0;
    }
    // two blocks at a time through the warp's [32 tokens][32 channels], 16-byte pieces permuted by the row
#pragma unroll
    for (int i0 = 0; i0 < B; i0 += 2) {
#pragma unroll
        for (int i = i0; i < i0 + 2; ++i) {
          const int n = n0 + 16 * i;
          uint32_t o[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float2 v = make_float2(sum[i][2 * j], sum[i][2 * j + 1]);
            if (bias) {
              v.x += n + 2 * j < p.N ? Elem<T>::to_float(bias[n + 2 * j]) : 0.f;
              v.y += n + 2 * j + 1 < p.N ? Elem<T>::to_float(bias[n + 2 * j + 1]) : 0.f;
            }
            o[j] = Elem<T>::pack(v.x, v.y);
          }
#pragma unroll
          for (int q = 0; q < 2; ++q)
            *reinterpret_cast<uint4*>(stage + lane * 64 + (((2 * (i - i0) + q) ^ (lane >> 1 & 3)) << 4)) =
                make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        }
        __syncwarp();
        const int n = n0 + 16 * i0;
        if (p.vec) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int r = 8 * q + (lane >> 2), c = lane & 3, at = m0 + 32 * quarter + r;
            const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 64 + ((c ^ (r >> 1 & 3)) << 4));
            if (at < p.M && n + 8 * c < p.N) *reinterpret_cast<uint4*>(y + (int64_t)at * p.N + n + 8 * c) = v;
          }
        } else {
          for (int r = 0; r < 32; ++r) {
            const int at = m0 + 32 * quarter + r;
            const uint16_t v = *reinterpret_cast<const uint16_t*>(stage + r * 64 + (((lane >> 3) ^ (r >> 1 & 3)) << 4) + 2 * (lane & 7));
            if (at < p.M && n + lane < p.N) reinterpret_cast<uint16_t*>(y)[(int64_t)at * p.N + n + lane] = v;
          }
        }
        __syncwarp();
      }
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowsThreads, 1)
    f8_rows_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap wmap2,
                   const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap smap, const F8Rows p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + p.park);   // the leader's, for both CTAs' copies
  uint64_t* empty = full + kRowsStages;
  uint64_t* acc_full = empty + kRowsStages;                      // [turn][half]
  uint64_t* acc_empty = acc_full + 4;                            // the leader's
  uint32_t* slot = reinterpret_cast<uint32_t*>(acc_empty + 4);
  uint8_t* scales = ring + p.park + kRowsBarriers;   // [stages + 2][128 tokens]: the epilogue is up to two stages behind the MMAs
  uint8_t* staging = scales + (kRowsStages + 2) * 512;
  const int warp = threadIdx.x >> 5;
  const int h0 = first_half(p.bn), h1 = p.bn - h0;               // channels of the two accumulators
  const int stage_bytes = kWBytes + p.bn / 2 * kChunk, St = p.stages;
  const int rank = (int)cluster_rank(), first = blockIdx.x / 2, step = gridDim.x / 2;

  if (threadIdx.x == 0) {
    for (int i = 0; i < St; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 2);   // both halves' MMAs
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 8);   // four warps of each CTA
    }
    mbar_fence_init();
  }
  if (warp == 1) tc::alloc_pair(slot, 512);
  tc::fence_before();
  cluster_sync_all();   // the peer's barriers exist before a copy or a commit reaches them
  tc::fence_after();
  const uint32_t tmem = *slot;
  pdl_launch_dependents();

  // 128 x 72 + 256 x 216 registers are the launch's 384 x 168: an epilogue thread holds 128 sums
  if (warp < 4) {
    tc::regs_dec<72>();
    if (warp == 0 || warp == 3) {
      // Two loaders, of the tokens and of the weights, as one would need longer for a stage than its MMAs take. The weights' first
      // stages do not wait for the kernel before.
      const bool weights = warp == 3;
      if (tc::elect_one()) {
        tma_prefetch_map(weights ? &wmap : &qmap);
        tma_prefetch_map(weights ? &wmap2 : &smap);
        const uint32_t bars = smem_addr(full), leader = mapa_shared(bars, 0);
        constexpr uint32_t kEmpty = 8 * kRowsStages;
        uint32_t dst = smem_addr(ring) + (weights ? kWBytes : 0), off = 0, phase = 1;   // of the stage; the ring starts out free
        const uint32_t dst0 = dst, off_end = 8 * St, expect = 2 * (stage_bytes + 512);
        uint32_t sdst = smem_addr(scales);
        const uint32_t sdst0 = sdst, sdst_end = sdst + 512 * (St + 2);
        int filled = 0;   // stages, up to the ring's
        bool ok = true, ready = false;
        if (!weights) pdl_wait();
        for (int tile = first; tile < p.tiles && ok; tile += step) {
          const TilePlace at = tile_place(tile, p.tiles_m, p.tiles_n);
          const int row = weights ? at.n * p.bn + h0 / 2 * rank : at.m * 256 + 128 * rank, row2 = at.n * p.bn + h0 + h1 / 2 * rank;
          for (int c = 0; c < p.chunks; ++c) {
            if (!ready) ok = wait_ready(bars + off + kEmpty, phase, &g_f8_status);
            if (!ok) break;
            if (weights) {
              tc::tma_load_2d_pair_at(dst, &wmap, c * kChunk, row, leader + off);
              tc::tma_load_2d_pair_at(dst + h0 / 2 * kChunk, &wmap2, c * kChunk, row2, leader + off);
            } else {
              if (rank == 0) mbar_arrive_expect_tx(&full[off / 8], expect);
              tc::tma_load_2d_pair_at(dst, &qmap, c * kChunk, row, leader + off);
              tc::tma_load_2d_pair_at(sdst, &smap, row, c, leader + off);
              sdst += 512;
              if (sdst == sdst_end) sdst = sdst0;
            }
            filled += filled < St;
            dst += stage_bytes;
            off += 8;
            if (off == off_end) off = 0, dst = dst0, phase ^= 1;
            ready = test_barrier(bars + off + kEmpty, phase);
          }
        }
        // no copy in flight past this point (the leader's barriers count all four loaders' copies): the stage to be filled next holds
        // the oldest of the last ones, its parity is that of its release before, and in a ring that was not filled the first does
        if (rank == 0 && !weights) {
          if (filled < St) off = 0, phase = 1;
          for (int k = 0; k < filled; ++k) {
            wait_ready(bars + off, phase ^ (filled < St), &g_f8_status);
            off += 8;
            if (off == off_end) off = 0, phase ^= 1;
          }
        }
      }
      __syncwarp();
    } else if (warp < 3) {
      // A warp a half of the channels, one lane running its whole loop. An instruction costs it some ten clocks, since it shares
      // its scheduler with epilogue warps and descriptors go through uniform registers: one lane for both halves took 1000
      // clocks a stage.
      const int h = warp - 1;
      if (rank == 0 && tc::elect_one()) {
        const uint32_t idesc = (1u << 4) | ((uint32_t)((h ? h1 : h0) >> 3) << 17) | ((256u >> 4) << 24);   // fp32 from e4m3, both K-major
        const uint32_t stage_step = (uint32_t)stage_bytes >> 4, b_off = (uint32_t)(kWBytes + h * (h0 / 2 * kChunk)) >> 4;
        const uint32_t desc0 = (uint32_t)tc::desc_sw128(smem_addr(ring), 16, 1024);   // counts 16 bytes
        const uint32_t bars = smem_addr(full), bar_end = bars + 8 * St, acc_bars = smem_addr(acc_full) + 8 * h, d0 = tmem + 128 * h;
        constexpr uint32_t kEmpty = 8 * kRowsStages, kAccEmpty = 32;   // bytes from a stage's or an accumulator's barrier to the other
        uint32_t ad = desc0, bar = bars, phase = 0, u = 0;            // of the stage; stages so far
        bool ready = false, free = true;   // (the first two accumulators are)
        const uint32_t mine = first < p.tiles ? (uint32_t)((p.tiles - first + step - 1) / step) * p.chunks : 0;
        for (; u < mine; ++u) {
          const uint32_t acc = acc_bars + 16 * (u & 1), d = d0 + 256 * (u & 1);
          if (!free && !wait_ready(acc + kAccEmpty, ((u >> 1) - 1) & 1, &g_f8_status)) break;
          if (!ready && !wait_ready(bar, phase, &g_f8_status)) break;
          tc::fence_after();
          const uint32_t b = ad + b_off;
          tc::mma_f8_ss_pair<false>(d, ad, b, idesc);
          tc::mma_f8_ss_pair<true>(d, ad + 2, b + 2, idesc);
          tc::mma_f8_ss_pair<true>(d, ad + 4, b + 4, idesc);
          tc::mma_f8_ss_pair<true>(d, ad + 6, b + 6, idesc);
          tc::commit_pair_at(acc);
          tc::commit_pair_at(bar + kEmpty);
          ad += stage_step;
          bar += 8;
          if (bar == bar_end) bar = bars, ad = desc0, phase ^= 1;
          // the next accumulator and stage, asked together
          free = u == 0 || test_barrier(acc_bars + kAccEmpty + 16 * (~u & 1), ((u + 1) / 2 - 1) & 1);
          ready = test_barrier(bar, phase);
        }
        // no MMA in flight past this point
        for (uint32_t i = 0; i < 2; ++i) {
          const uint32_t uses = (u + 1 - i) >> 1;
          if (uses > 0) wait_ready(acc_bars + 16 * i, (uses - 1) & 1, &g_f8_status);
        }
      }
      __syncwarp();
    }
  } else {
    tc::regs_inc<216>();
    const int e = warp - 4, h = e >> 2;
    const F8Epilogue w{smem_addr(acc_full), mapa_shared(smem_addr(acc_empty), 0), smem_addr(scales), tmem, staging + e * kRowsSmem, rank, first, step, h0 * h, h};
    const int blocks = (h ? h1 : h0) / 16;
    pdl_wait();
    blocks == 8 ? rows_epilogue<T, 8>(p, w) : blocks == 6 ? rows_epilogue<T, 6>(p, w) : blocks == 4 ? rows_epilogue<T, 4>(p, w) : rows_epilogue<T, 2>(p, w);
  }
  __syncwarp();
  tc::fence_before();
  cluster_sync_all();   // neither CTA leaves while its partner still signals its shared memory
  if (warp == 1) {
    tc::fence_after();
    tc::dealloc_pair(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------------------- the product, one to eight tokens
// A CTA takes 16 channels and all of K: mma.sync m16n8k32 with the weights' fragments loaded straight into registers, 64 bytes
// of K (half a block) of a row per four lanes and 16-byte load (the order of k inside a fragment is free as long as both
// operands share it); each piece's sums are scaled into fp32 registers. The first loads are issued at once, with `early` before
// the wait on the previous kernel; the CTA quantizes the token rows while they are under way. On this
// machine mma.sync takes e4m3 by converting it to fp16, which is a third of the instructions. One token, cold weights: 2048 x
// 11008 7.8 us (6.2 without the quantization, in a graph with the call before still running 6.0), 1536 x 8960 4.7, 3584 x 3584
// 5.2. (fp16 tokens in shared memory, converted once: 8.3, 5.4, 6.0; scales of the weights fetched with them: 8.5, 4.9, 5.5.)
constexpr int kGemvRows = 8;

struct F8Gemv {
  const void* x;
  int64_t ldx;
  const uint8_t* w;
  int64_t ldw;
  const float* t;
  const void* bias;
  void* y;
  int M, N, K, blocks;
  int pitch;             // bytes between the quantized rows: 64 modulo 128, so that two rows' reads do not share banks
};

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// MR: the most rows, 1, 4 or 8. R: 64-byte pieces of K a warp has in flight. An SM holds gemv_per_sm of its CTAs.
constexpr int gemv_per_sm(int NW, int MR, int R) {
  return NW == 16 ? (R == 2 && MR < 8 ? 2 : 1) : (MR == 8 ? 2 : 3) + (R == 2);
}
template <typename T, int NW, int MR, int R>
__global__ void __launch_bounds__(32 * NW, gemv_per_sm(NW, MR, R)) f8_gemv_kernel(const F8Gemv p, bool early) {
  extern __shared__ __align__(16) uint8_t rows[];   // [M][pitch] quantized tokens, then the scales s t [blocks][MR]
  __shared__ float part[NW][128];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16, pieces = 2 * p.blocks;
  float* scales = reinterpret_cast<float*>(rows + p.M * p.pitch);
  pdl_launch_dependents();
  if (!early) pdl_wait();
  // rows past N repeat the last one; pieces past K read as zeros (K is padded to 16, a lane's share of a piece)
  const uint8_t* w0 = p.w + (int64_t)min(n0 + g, p.N - 1) * p.ldw + 16 * t;
  const uint8_t* w1 = p.w + (int64_t)min(n0 + g + 8, p.N - 1) * p.ldw + 16 * t;
  const float* tb = p.t + (int64_t)(n0 / kBlock) * p.blocks;
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
  if (early) pdl_wait();
  const bool aligned = ((reinterpret_cast<uintptr_t>(p.x) | (uintptr_t)(p.ldx * sizeof(T))) & 15u) == 0;
  const T* x = static_cast<const T*>(p.x);
  // 16 lanes a block of 128 values; all rows' loads of a round under way together
  for (int j0 = 0; j0 < 16 * p.blocks; j0 += 32 * NW) {
    const int j = j0 + tid;
    const float t128 = (j & 15) == 0 && j < 16 * p.blocks ? __ldcg(tb + (j >> 4)) : 0.f;
    uint4 v[MR];
#pragma unroll
    for (int m = 0; m < MR; ++m)
      v[m] = m < p.M && 8 * j < p.K ? load8(x + m * p.ldx + 8 * j, p.K - 8 * j, aligned) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int m = 0; m < MR; ++m)
      if (m < p.M) {
        float f[8];
        floats8<T>(v[m], f);
        uint32_t am = amax_packed<T>(v[m]);
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) am = max(am, __shfl_xor_sync(0xffffffffu, am, d));
        const BlockScale sc = block_scale(am);
        if (j < 16 * p.blocks) {
          *reinterpret_cast<uint2*>(rows + m * p.pitch + 8 * j) = e4m3x8(f, sc.up);
          if ((j & 15) == 0) scales[(j >> 4) * MR + m] = sc.s * t128;
        }
      }
  }
  __syncthreads();
  // behind the wait, since the kernel before may have written it, and on its way under the products
  const uint16_t bias = out_on && p.bias ? ldg_cg_u16(static_cast<const T*>(p.bias) + out_n) : (uint16_t)0;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  const uint32_t own = smem_addr(rows) + (uint32_t)(min(g, p.M - 1) * p.pitch + 16 * t);   // unused columns repeat a row
  const int m0 = min(2 * t, p.M - 1), m1 = min(2 * t + 1, p.M - 1);
  for (int c0 = warp; c0 < pieces; c0 += NW * R) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = c0 + i * NW;
      if (c < pieces) {
        const uint4 b = lds128(own + 64 * c);
        const float s0 = scales[(c >> 1) * MR + m0], s1 = scales[(c >> 1) * MR + m1];
        float d[4] = {0.f, 0.f, 0.f, 0.f};
        mma_e4m3(d, a[i][0].x, a[i][1].x, a[i][0].y, a[i][1].y, b.x, b.y);
        mma_e4m3(d, a[i][0].z, a[i][1].z, a[i][0].w, a[i][1].w, b.z, b.w);
        fetch(i, c + NW * R);
        sum[0] = fmaf(d[0], s0, sum[0]);
        sum[1] = fmaf(d[1], s1, sum[1]);
        sum[2] = fmaf(d[2], s0, sum[2]);
        sum[3] = fmaf(d[3], s1, sum[3]);
      }
    }
  }
  // D[g][2t], D[g][2t + 1], D[g + 8][..]: channel x token
  part[warp][(2 * t) * 16 + g] = sum[0];
  part[warp][(2 * t + 1) * 16 + g] = sum[1];
  part[warp][(2 * t) * 16 + g + 8] = sum[2];
  part[warp][(2 * t + 1) * 16 + g + 8] = sum[3];
  __syncthreads();
  if (out_on) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += part[w][tid];
    static_cast<T*>(p.y)[(int64_t)out_m * p.N + out_n] = Elem<T>::from_float(v + Elem<T>::unpack(bias).x);
  }
}

// ------------------------------------------------------------------------------------------------------- launches
template <typename Kern, typename... Args>
cudaError_t launch_f8(Kern kern, dim3 grid, int threads, size_t smem, int cluster, bool pdl, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
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
cudaError_t allow_smem(Kern kern, std::atomic<uint64_t>& done, int bytes = kSmem) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

int64_t padded(int64_t k) { return (k + 15) / 16 * 16; }
int64_t blocks_of(int64_t k) { return (k + kBlock - 1) / kBlock; }
int64_t scale_rows(int64_t m) { return (m + 3) / 4 * 4; }

bool encode_rows(CUtensorMap* map, const void* base, int64_t width, int64_t ld, int64_t rows, int box_rows) {
  return encode_tensor_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, (uint64_t)width, (uint64_t)rows, (uint64_t)ld, kChunk,
                              (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

int tmem_columns(int bn) { return bn <= 32 ? 32 : bn <= 64 ? 64 : 128; }

// Which side the tokens are, the other side's width, K split and stages: the candidate whose estimated time is least, in clocks
// per CTA: a start and an end; per wave and stage what the way of an accumulator costs beside its columns (fitted to the
// product at bn = 128 to 256: 8192 x 18944 x 3584, 4096 x 4096 x 3584; and 61 to 300 tokens of 3584, both sides' kernels: 129
// tokens of 4608 channels 16.7 / 18.0 us, 257 22.4 / 20.1); stores; and a cluster's sum where all its CTAs can be resident.
struct F8Plan {
  int bn, splits, stages;
  bool rows;   // tokens as the A side, a pair of CTAs a tile
};

template <typename T, int NB>
int resident_clusters(int S) {   // of S single CTAs with the whole shared memory each, on the current device
  static std::atomic<int> known[64][kMaxSplits + 1];
  int dev = 0;
  cudaGetDevice(&dev);
  std::atomic<int>& k = known[dev & 63][S];
  int v = k.load(std::memory_order_relaxed);
  if (v == 0) {
    static std::atomic<uint64_t> done{0};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S);
    cfg.blockDim = dim3(kMmaThreads);
    cfg.dynamicSmemBytes = kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = S;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (allow_smem(f8_cols_kernel<T, NB>, done) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, f8_cols_kernel<T, NB>, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    v = n + 1;
    k.store(v, std::memory_order_relaxed);
  }
  return v - 1;
}

template <typename T>
F8Plan f8_plan(int64_t M, int64_t N, int chunks, int sms) {
  F8Plan best{0, 1, 0, false};
  int64_t least = INT64_MAX;
  auto consider = [&](int bn, bool rows, int S) {
    const int64_t tiles = rows ? (M + 255) / 256 * ((N + bn - 1) / bn) : (M + bn - 1) / bn * ((N + 127) / 128);
    if (S > 1 && tiles > resident_clusters<T, 2>(S)) return;
    const int64_t ctas = tiles * (rows ? 2 : S), waves = (ctas + sms - 1) / sms;
    const int64_t chunk = rows ? 600 + 2 * bn : 700 + 3 * bn;
    const int64_t c = 4700 + waves * ((chunks + S - 1) / S) * chunk + waves * 8 * bn + (S > 1 ? 2800 : 0);
    if (c < least) {
      least = c;
      best.bn = bn, best.rows = rows, best.splits = S;
    }
  };
  for (int bn = 256; bn >= 64; bn -= 32) consider(bn, true, 1);
  for (int bn = 128; bn >= 16; bn -= 16) {
    if (bn - 16 >= M) continue;   // wider than the tokens
    for (int S = 1; S <= kMaxSplits && (S == 1 || chunks >= 2 * S); ++S) consider(bn, false, S);
  }
  best.stages = min(best.rows ? kRowsStages : kMaxStages, (kSmem - 1024 - (best.rows ? kRowsBarrierBytes : kBarrierBytes)) /
                                    (kWBytes + (best.rows ? best.bn / 2 : best.bn) * kChunk));
  return best;
}

// Blocks a CTA: two where the product starts beside the quantization; behind it one, until that makes many CTAs (QB = 1, 2, 4:
// 100 x 8960 x 1536 14.3, 13.8, 15.1 us; 61 x 18944 x 3584 24.1, 24.2, 24.7; 300 x 3584 x 4608 18.8, 19.3, 21.0; 1000 x 1536 x 2048 12.4,
// 13.3, 15.1; 2048 x 18944 x 3584 169.6, 168.0, 167.6; 8192 x 18944 x 3584 670, 672, 636; 61 x 3584 x 4608 13.2 with each)
template <typename T>
cudaError_t tokens_t(const void* x, int64_t ldx, uint8_t* q, int64_t ldq, float* s, int64_t lds, int64_t M, int64_t K, int release,
                     bool pdl, cudaStream_t st) {
  const int64_t blocks = blocks_of(K), rows = (M + 15) / 16;
  const int per = release != kAtEnd ? 2 : blocks * rows <= 8192 ? 1 : 4;
  auto kern = per == 1 ? f8_tokens_kernel<T, 1> : per == 2 ? f8_tokens_kernel<T, 2> : f8_tokens_kernel<T, 4>;
  return launch_f8(kern, dim3((unsigned)((blocks + per - 1) / per), (unsigned)rows), 256, 0, 1, pdl, st, static_cast<const T*>(x), ldx, q,
                   (int)ldq, s, (int)lds, (int)M, (int)K, release);
}

template <typename T, int NB>
cudaError_t cols_t(const CUtensorMap& wmap, const CUtensorMap& qmap, const F8Gemm& g, size_t smem, int sms, bool pdl, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(f8_cols_kernel<T, NB>, done);
  if (e != cudaSuccess) return e;
  return launch_f8(f8_cols_kernel<T, NB>, dim3((unsigned)(g.splits > 1 ? g.tiles * g.splits : min(g.tiles, sms))), kMmaThreads, smem,
                   g.splits, pdl, st, wmap, qmap, g);
}

// One to eight tokens, while their values are few: every CTA quantizes all of them. The bound is the one of the 8-bit integer product,
// not fitted to this one. One launch / two, us, cold weights: inside it 4 x 2048 x 11008 9.9 / 13.5, 8 x 1536 x 4608 5.4 / 8.8; outside it
// narrow layers would still gain (4 x 3584 x 4608 6.5 / 11.0, 2 x 8960 x 1536 6.8 / 10.5, 3 x 11008 x 2048 8.8 / 12.6), others would not
// (8 x 3584 x 3584 10.0 / 10.0, 1 x 18944 x 3584 20.4 / 20.6, 2 x 18944 x 3584 23.6 / 20.8, 4 x 3584 x 18944 25.5 / 19.4).
bool gemv_takes(int64_t M, int64_t K) { return M <= kGemvRows && M * K <= 12288; }

template <typename T>
cudaError_t gemv_t(const F8Params& p, bool pdl, cudaStream_t st) {
  const int blocks = (int)blocks_of(p.K), pitch = blocks * kBlock + 64, mr = p.M == 1 ? 1 : p.M <= 4 ? 4 : 8;
  const F8Gemv g{p.x, p.ldx, static_cast<const uint8_t*>(p.w), p.ldw, p.w_scales, p.bias, p.y, (int)p.M, (int)p.N, (int)p.K, blocks, pitch};
  // 8 warps where they hold all of K, on wide layers; else 16. R = 4, or R = 2 where the more CTAs an SM then holds save a round
  const int warps = blocks > 16 || p.N < 4096 ? 16 : 8, ctas = (int)((p.N + 15) / 16), sms = sm_count();
  auto rounds = [&](int per) { return (ctas + per * sms - 1) / (per * sms); };
#define LB_GEMV(MR)                                                                                                   \
  (warps == 8 ? (rounds(gemv_per_sm(8, MR, 2)) < rounds(gemv_per_sm(8, MR, 4)) ? f8_gemv_kernel<T, 8, MR, 2>           \
                                                                               : f8_gemv_kernel<T, 8, MR, 4>)          \
              : (rounds(gemv_per_sm(16, MR, 2)) < rounds(gemv_per_sm(16, MR, 4)) ? f8_gemv_kernel<T, 16, MR, 2>        \
                                                                                 : f8_gemv_kernel<T, 16, MR, 4>))
  auto kern = p.M == 1 ? LB_GEMV(1) : p.M <= 4 ? LB_GEMV(4) : LB_GEMV(8);
#undef LB_GEMV
  return launch_f8(kern, dim3((unsigned)ctas), 32 * warps, (size_t)p.M * pitch + (size_t)blocks * mr * 4, 1, pdl, st, g, p.early);
}

template <typename T>
cudaError_t linear_t(const F8Params& p, bool pdl, cudaStream_t st) {
  if (gemv_takes(p.M, p.K)) return gemv_t<T>(p, pdl, st);
  const int sms = sm_count();
  const int64_t kp = padded(p.K), lds = scale_rows(p.M);
  const int chunks = (int)blocks_of(p.K);
  uint8_t* q = static_cast<uint8_t*>(p.workspace);
  float* s = reinterpret_cast<float*>(q + p.M * kp);
  // with few rows the product is let in early, see lb_w8.cu: it may read weights before it waits, so where they may still be
  // in the making only once everything before the quantization is complete
  const Release release = p.M > 296 ? kAtEnd : p.early ? kAtEntry : kAfterWait;
  cudaError_t e = tokens_t<T>(p.x, p.ldx, q, kp, s, lds, p.M, p.K, release, pdl, st);
  if (e != cudaSuccess) return e;
  static thread_local struct {   // the last plan of this host thread, for calls of one shape that follow one another
    int64_t M, N, chunks;
    int sms;
    F8Plan plan;
  } last = {};
  if (last.M != p.M || last.N != p.N || last.chunks != chunks || last.sms != sms)
    last = {p.M, p.N, chunks, sms, f8_plan<T>(p.M, p.N, chunks, sms)};
  const F8Plan plan = last.plan;
  CUtensorMap wmap, qmap;
  const bool vec = p.N % 8 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15u) == 0;
  const int tile_m = plan.rows ? 256 : plan.bn, tile_n = plan.rows ? plan.bn : 128;
  const int tiles_m = (int)((p.M + tile_m - 1) / tile_m), tiles = (int)((p.N + tile_n - 1) / tile_n) * tiles_m;
  if (plan.rows) {
    CUtensorMap wmap2, smap;
    const int h0 = first_half(plan.bn);
    if (!encode_rows(&wmap, p.w, kp, p.ldw, p.N, h0 / 2) || !encode_rows(&wmap2, p.w, kp, p.ldw, p.N, (plan.bn - h0) / 2) ||
        !encode_rows(&qmap, q, kp, kp, p.M, 128) ||
        !encode_tensor_map_2d(&smap, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, s, (uint64_t)lds, (uint64_t)chunks, (uint64_t)lds * 4, 128, 1, CU_TENSOR_MAP_SWIZZLE_NONE))
      return cudaErrorInvalidValue;
    const int park = plan.stages * (kWBytes + plan.bn / 2 * kChunk);
    const F8Rows g{p.w_scales, p.bias, p.y, (int)p.M, (int)p.N, chunks, plan.bn, tiles_m, tiles / tiles_m, tiles, plan.stages, park, vec};
    static std::atomic<uint64_t> done{0};
    if ((e = allow_smem(f8_rows_kernel<T>, done)) != cudaSuccess) return e;
    return launch_f8(f8_rows_kernel<T>, dim3((unsigned)(2 * min(tiles, sms / 2))), kRowsThreads, (size_t)park + kRowsBarrierBytes + 1024, 2, pdl,
                     st, wmap, wmap2, qmap, smap, g);
  }
  if (!encode_rows(&wmap, p.w, kp, p.ldw, p.N, 128) || !encode_rows(&qmap, q, kp, kp, p.M, plan.bn)) return cudaErrorInvalidValue;
  const int stride = tmem_columns(plan.bn), park = plan.stages * (kWBytes + plan.bn * kChunk);
  const F8Gemm g{s, p.w_scales, p.bias, p.y, (int)p.M, (int)p.N, chunks, (int)lds, plan.bn, tiles_m, tiles, plan.splits, plan.stages,
                 min(kMaxAcc, 512 / stride), stride, park, vec};
  const size_t smem = (size_t)park + kBarrierBytes + 1024;
  return plan.bn <= 64 ? cols_t<T, 1>(wmap, qmap, g, smem, sms, pdl, st) : cols_t<T, 2>(wmap, qmap, g, smem, sms, pdl, st);
}

}  // namespace

// none where the product quantizes by itself
size_t f8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (gemv_takes(M, K)) return 0;
  return (size_t)M * (size_t)padded(K) + (size_t)scale_rows(M) * blocks_of(K) * 4;
}

cudaError_t launch_f8_quantize_weight(const void* w, int dtype, int64_t ldw, void* q, int64_t ldq, float* t, int64_t N, int64_t K,
                                      bool pdl, cudaStream_t st) {
  const dim3 grid((unsigned)blocks_of(K), (unsigned)blocks_of(N));
  uint8_t* out = static_cast<uint8_t*>(q);
  return dtype == 0   ? launch_f8(f8_weight_kernel<__half>, grid, 256, 0, 1, pdl, st, static_cast<const __half*>(w), ldw, out, ldq, t, (int)N, (int)K)
         : dtype == 1 ? launch_f8(f8_weight_kernel<__nv_bfloat16>, grid, 256, 0, 1, pdl, st, static_cast<const __nv_bfloat16*>(w), ldw, out, ldq, t, (int)N, (int)K)
                      : launch_f8(f8_weight_kernel<float>, grid, 256, 0, 1, pdl, st, static_cast<const float*>(w), ldw, out, ldq, t, (int)N, (int)K);
}

cudaError_t launch_f8_linear(const F8Params& p, bool pdl, cudaStream_t st) {
  return p.dtype == 0 ? linear_t<__half>(p, pdl, st) : linear_t<__nv_bfloat16>(p, pdl, st);
}

int f8_device_error() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_f8_status, sizeof(int));
  return v;
}

void f8_clear_device_error() {
  int z = 0;
  cudaMemcpyToSymbol(g_f8_status, &z, sizeof(int));
}

}  // namespace lb
