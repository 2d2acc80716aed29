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

// Tokens: 16 lanes take a block of 128 values, a warp two tokens, a CTA 16 tokens x kQBlocks blocks, all of whose loads are
// under way at once. The scales go to [block][token], as the product reads them, 16 tokens a run. Bound by memory.
constexpr int kQBlocks = 4;
enum Release { kAtEnd, kAfterWait, kAtEntry };   // when the quantization lets the next kernel start

template <typename T>
__global__ void __launch_bounds__(256)
    f8_tokens_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, int ldq, float* __restrict__ s, int lds,
                     int M, int K, int release) {
  if (release == kAtEntry) pdl_launch_dependents();
  pdl_wait();
  if (release == kAfterWait) pdl_launch_dependents();
  const int g = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int m = blockIdx.y * 16 + g, b0 = blockIdx.x * kQBlocks;
  const bool aligned = ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(ldx * sizeof(T))) & 15u) == 0;
  const T* row = x + (int64_t)min(m, M - 1) * ldx;
  uint4 v[kQBlocks];
#pragma unroll
  for (int i = 0; i < kQBlocks; ++i) {
    const int k = (b0 + i) * kBlock + 8 * lane;
    v[i] = k < K ? load8(row + k, K - k, aligned) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < kQBlocks; ++i) {
    const int b = b0 + i, k = b * kBlock + 8 * lane;
    float f[8];
    floats8<T>(v[i], f);
    uint32_t a = amax8(f);
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

// ------------------------------------------------------------------------------------------------------- the product
// tcgen05.mma kind::f8f6f4 with the channels as the A side (128 a CTA, which is a row of the weights' blocks) and a tile of
// bn tokens as the N side. A stage of the ring is 128 bytes of K, so one block of the scales: each stage's four MMAs start a
// new accumulator, and 16 epilogue warps add it, times s t, to the sums that they hold in registers (a lane a channel, a
// column a token) while the next stages' MMAs run into the other accumulators. The scale of a column is the same for all
// lanes: each warp puts its columns' s t into shared memory, from where four come in one broadcast load; two columns take
// one fp32-pair multiply-add.
// PAIR: two CTAs work on one tile of 256 channels (cta_group::2): each loads its 128 channels and half of the tokens.
// CTAs are persistent over tiles, tokens innermost. Few tiles and long K: a cluster of S single CTAs splits K, each parks
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

template <typename T, bool PAIR, int NB>   // NB: 16-column blocks of a tile a warp holds, bn <= 64 NB
__global__ void __launch_bounds__(kMmaThreads, 1)
    f8_gemm_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap qmap, const F8Gemm p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + p.park);   // PAIR: the leader's, for both CTAs' copies
  uint64_t* empty = full + kMaxStages;
  uint64_t* acc_full = empty + kMaxStages;
  uint64_t* acc_empty = acc_full + kMaxAcc;                      // PAIR: the leader's
  uint32_t* slot = reinterpret_cast<uint32_t*>(acc_empty + kMaxAcc);
  float* scales = reinterpret_cast<float*>(slot + 4);            // [epilogue warps][2][64]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int own_bn = PAIR ? p.bn / 2 : p.bn;                     // tokens this CTA loads
  const int stage_bytes = kWBytes + own_bn * kChunk, S = PAIR ? 1 : p.splits, St = p.stages, A = p.acc;
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
    for (int i = 0; i < A; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], PAIR ? 2 * kEpiWarps : kEpiWarps);
    }
    mbar_fence_init();
  }
  const uint32_t columns = (uint32_t)(A * p.acc_stride);
  if (warp == 1) {
    if (PAIR)
      tc::alloc_pair(slot, columns);
    else
      tc::alloc(slot, columns);
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
      struct Place {
        int tile, c, m0, n0;
      };
      auto at = [&](int tile) {
        const int n = tile / p.tiles_m, m = tile - n * p.tiles_m;
        return Place{tile, 0, m * p.bn + (PAIR ? rank * own_bn : 0), n * kTileN + n_off};
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
          tc::tma_load_2d_pair(dst, &qmap, q.c * kChunk, q.m0, mapa_shared(smem_addr(&full[s]), 0));
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
        ok = wait_bounded(&empty[s], phase, &g_f8_status);
        if (!ok) break;
        weights(q, s);
        tokens(q, s);
        if (++s == St) s = 0, phase ^= 1;
      }
      // no copy in flight past this point (a pair's leader's barriers count its peer's copies too): stage s holds the
      // oldest of the last `head` copies, its parity is that of the release before it
      if (rank == 0 || !PAIR)
        for (int i = 0; i < head; ++i) {
          wait_bounded(&full[s], phase, &g_f8_status);
          if (++s == head) s = 0, phase ^= 1;
        }
    }
    __syncwarp();
  } else if (warp == 1) {
    if ((!PAIR || rank == 0) && tc::elect_one()) {
      // fp32 accumulator, e4m3 A and B, both K-major
      const uint32_t idesc = (1u << 4) | ((uint32_t)(p.bn >> 3) << 17) | ((uint32_t)(kTileN >> 4) << 24);
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
          for (int k = 0; k < 4; ++k) {
            if (PAIR)
              tc::mma_f8_ss_pair(d, ad + 2 * k, bd + 2 * k, idesc, k > 0);
            else
              tc::mma_f8_ss(d, ad + 2 * k, bd + 2 * k, idesc, k > 0);
          }
          if (PAIR) {
            tc::commit_pair(&empty[s]);
            tc::commit_pair(&acc_full[a]);
          } else {
            tc::commit(&empty[s]);
            tc::commit(&acc_full[a]);
          }
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
      const int m0 = tile % p.tiles_m * p.bn, nt = tile / p.tiles_m, n = nt * kTileN + n_off + row;
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
      const float* tp = p.t + (int64_t)min((nt * kTileN + n_off) / kBlock, (p.N - 1) / kBlock) * p.chunks + c0;
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
        if (lane == 0) {
          if (PAIR)
            tc::arrive_cluster(mapa_shared(smem_addr(&acc_empty[a]), 0));
          else
            mbar_arrive(&acc_empty[a]);
        }
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
  if (!PAIR && S > 1) {
    const int n0 = first / p.tiles_m * 128, m0 = first % p.tiles_m * p.bn;
    sum_partials<T>(smem_addr(ring), static_cast<const T*>(p.bias), static_cast<T*>(p.y) + (int64_t)m0 * p.N, n0, p.N,
                    min(p.bn, p.M - m0), rank, S);
  }
  tc::fence_before();
  if (PAIR || S > 1)
    cluster_sync_all();   // no CTA leaves while its partner still reads, or signals, its shared memory
  else
    __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    if (PAIR)
      tc::dealloc_pair(tmem, columns);
    else
      tc::dealloc(tmem, columns);
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

int tmem_columns(int bn) { return bn <= 32 ? 32 : bn <= 64 ? 64 : bn <= 128 ? 128 : 256; }

// Tokens per tile, pairs or single CTAs, K split and stages: the candidate whose estimated time is least, in clocks per
// CTA.
struct F8Plan {
  int bn, splits, stages;
  bool pair;
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
    if (allow_smem(f8_gemm_kernel<T, false, NB>, done) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, f8_gemm_kernel<T, false, NB>, &cfg) != cudaSuccess) {
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
  auto consider = [&](int bn, bool pair, int S) {
    const int64_t tiles = (M + bn - 1) / bn * (pair ? (N + 255) / 256 : (N + 127) / 128);
    if (S > 1 && tiles > resident_clusters<T, 4>(S)) return;
    const int64_t ctas = tiles * (pair ? 2 : S), waves = (ctas + sms - 1) / sms;
    const int64_t chunk = max(450, 2 * bn) + (kWBytes + (pair ? bn / 2 : bn) * kChunk) / 64;
    const int64_t c = 4700 + waves * ((chunks + S - 1) / S) * chunk + waves * 8 * bn + (S > 1 ? 2800 : 0);
    if (c < least) {
      least = c;
      best.bn = bn, best.pair = pair, best.splits = S;
    }
  };
  for (int bn = 256; bn >= 64; bn -= 32) consider(bn, true, 1);
  for (int bn = 256; bn >= 16; bn -= 16) {
    if (bn - 16 >= M) continue;   // wider than the tokens
    for (int S = 1; S <= kMaxSplits && (S == 1 || chunks >= 2 * S); ++S) consider(bn, false, S);
  }
  best.stages = min(kMaxStages, (kSmem - 1024 - kBarrierBytes) / (kWBytes + (best.pair ? best.bn / 2 : best.bn) * kChunk));
  return best;
}

template <typename T>
cudaError_t tokens_t(const void* x, int64_t ldx, uint8_t* q, int64_t ldq, float* s, int64_t lds, int64_t M, int64_t K, int release,
                     bool pdl, cudaStream_t st) {
  const dim3 grid((unsigned)((blocks_of(K) + kQBlocks - 1) / kQBlocks), (unsigned)((M + 15) / 16));
  return launch_f8(f8_tokens_kernel<T>, grid, 256, 0, 1, pdl, st, static_cast<const T*>(x), ldx, q, (int)ldq, s, (int)lds, (int)M,
                   (int)K, release);
}

template <typename T, bool PAIR, int NB>
cudaError_t gemm_t(const CUtensorMap& wmap, const CUtensorMap& qmap, const F8Gemm& g, unsigned ctas, size_t smem, bool pdl,
                   cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(f8_gemm_kernel<T, PAIR, NB>, done);
  if (e != cudaSuccess) return e;
  return launch_f8(f8_gemm_kernel<T, PAIR, NB>, dim3(ctas), kMmaThreads, smem, PAIR ? 2 : g.splits, pdl, st, wmap, qmap, g);
}

template <typename T>
cudaError_t linear_t(const F8Params& p, bool pdl, cudaStream_t st) {
  const int sms = sm_count();
  const int64_t kp = padded(p.K), lds = scale_rows(p.M);
  const int chunks = (int)blocks_of(p.K);
  uint8_t* q = static_cast<uint8_t*>(p.workspace);
  float* s = reinterpret_cast<float*>(q + p.M * kp);
  CUtensorMap wmap, qmap;
  if (!encode_rows(&wmap, p.w, kp, p.ldw, p.N, 128)) return cudaErrorInvalidValue;
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
  const int own_bn = plan.pair ? plan.bn / 2 : plan.bn, tile_n = plan.pair ? 256 : 128;
  const int tiles_m = (int)((p.M + plan.bn - 1) / plan.bn), tiles = (int)((p.N + tile_n - 1) / tile_n) * tiles_m;
  const int stride = tmem_columns(plan.bn), park = plan.stages * (kWBytes + own_bn * kChunk);
  const F8Gemm g{s, p.w_scales, p.bias, p.y, (int)p.M, (int)p.N, chunks, (int)lds, plan.bn, tiles_m, tiles, plan.splits, plan.stages,
                 min(kMaxAcc, 512 / stride), stride, park, p.N % 8 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15u) == 0};
  if (!encode_rows(&qmap, q, kp, kp, p.M, own_bn)) return cudaErrorInvalidValue;
  const size_t smem = (size_t)park + kBarrierBytes + 1024;
  if (plan.pair) {
    const unsigned ctas = (unsigned)(2 * min(tiles, sms / 2));
    return plan.bn <= 128 ? gemm_t<T, true, 2>(wmap, qmap, g, ctas, smem, pdl, st) : gemm_t<T, true, 4>(wmap, qmap, g, ctas, smem, pdl, st);
  }
  const unsigned ctas = (unsigned)(plan.splits > 1 ? tiles * plan.splits : min(tiles, sms));
  return plan.bn <= 64    ? gemm_t<T, false, 1>(wmap, qmap, g, ctas, smem, pdl, st)
         : plan.bn <= 128 ? gemm_t<T, false, 2>(wmap, qmap, g, ctas, smem, pdl, st)
                          : gemm_t<T, false, 4>(wmap, qmap, g, ctas, smem, pdl, st);
}

}  // namespace

size_t f8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
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
