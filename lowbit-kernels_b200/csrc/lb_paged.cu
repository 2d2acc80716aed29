// The paged KV cache: per-head norm + rotary rotation + append of a chunk of new tokens, and the attention of new
// tokens over the cache.
//
// Cache: K and V are [pages, nkv, page_size, hd], each page's block contiguous, pages a stride apart; a sequence's
// context lies in the pages its row of the page table lists, page_size tokens each.
#include <atomic>

#include "lb_launch.h"
#include "lb_tma.cuh"
#include "lb_types.cuh"

namespace lb {

// status word of this file's kernels: a bounded wait that gave up, or a slot or page outside the cache
__device__ int g_paged_status;

namespace {

// ------------------------------------------------------------------------------------------------------- append
// q and k heads: x <- x rsqrt(mean(x^2) + eps) w (where norm weights are given), then the pair (x_i, x_{i + F}),
// i < F, turned by the angle pos * f_i; the dimensions from 2F on are left as they are. v heads are copied. All in
// fp32, one rounding. Memory bound: each value is read once and written once.
//
// A group of G lanes takes one head of one token, 16 values a lane as two 16-byte vectors: lane j < F / 8 the vectors
// j and j + F / 8 (the two halves of eight pairs, so the rotation needs no exchange), the lanes after them two
// neighbouring vectors of the unrotated rest. A CTA holds whole tokens, whose cosines and sines it computes once in
// shared memory: the angle in fp64 as a multiple of pi (fp32 would lose 1e-3 of a turn at position 1e5), while the
// CTA's values are already on their way from memory.
constexpr int kAppendMaxThreads = 512;

struct AppendParams {
  const void* qkv;
  int64_t ld;       // elements between tokens
  int tokens, nh, nkv, hd, F;
  const void* q_norm;
  const void* k_norm;
  float eps;
  const float* inv_freq;
  const int64_t* pos;
  const int64_t* slots;
  void* q_out;      // [tokens, nh, hd]
  void* k;
  void* v;
  int64_t k_page, v_page;   // elements between pages
  int64_t num_slots;
  int page_size;
  int tpb;          // tokens per CTA
};

template <typename T, int G>
__global__ void __launch_bounds__(kAppendMaxThreads) append_kernel(const AppendParams p) {
  extern __shared__ float2 turn[];   // [tpb][F]: cos, sin
  pdl_launch_dependents();
  const int heads = p.nh + 2 * p.nkv, lanes = p.hd / 16, f8 = p.F / 8;
  const int t0 = blockIdx.x * p.tpb, nt = min(p.tpb, p.tokens - t0);
  const int lane = threadIdx.x % G, per = blockDim.x / G;
  const int v0 = lane < f8 ? lane : 2 * lane, v1 = lane < f8 ? lane + f8 : 2 * lane + 1;
  const bool on = lane < lanes;
  float wq[16], wk[16];
  const bool norm = p.q_norm != nullptr;
  if (norm && on) {   // model state: read before the wait
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = 8 * (h ? v1 : v0) + i;
        wq[8 * h + i] = Elem<T>::to_float(static_cast<const T*>(p.q_norm)[d]);
        wk[8 * h + i] = Elem<T>::to_float(static_cast<const T*>(p.k_norm)[d]);
      }
  }
  pdl_wait();
  const T* qkv = static_cast<const T*>(p.qkv);
  const int units = nt * heads;
  uint4 x[2];
  auto load = [&](int u) {
    if (u < units && on) {
      const T* src = qkv + (int64_t)(t0 + u / heads) * p.ld + (u % heads) * p.hd;
      x[0] = *reinterpret_cast<const uint4*>(src + 8 * v0);
      x[1] = *reinterpret_cast<const uint4*>(src + 8 * v1);
    }
  };
  load(threadIdx.x / G);
  for (int i = threadIdx.x; i < nt * p.F; i += blockDim.x) {
    // angle / pi reduced to [-1, 1] in fp64
    double a = (double)p.pos[t0 + i / p.F] * (double)p.inv_freq[i % p.F] * 0.31830988618379067154;
    a -= 2.0 * rint(a * 0.5);
    float sn, cs;
    sincospif((float)a, &sn, &cs);
    turn[i] = make_float2(cs, sn);
  }
  __syncthreads();
  for (int u0 = 0; u0 < units; u0 += per) {
    const int u = u0 + threadIdx.x / G;
    if (u0) load(u);
    const bool live = u < units && on;
    const int tl = u / heads, head = u % heads, t = t0 + tl;
    float f[16];
    const uint32_t* xw = reinterpret_cast<const uint32_t*>(x);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 a = live ? Elem<T>::unpack(xw[i]) : make_float2(0.f, 0.f);
      f[2 * i] = a.x;
      f[2 * i + 1] = a.y;
    }
    const bool is_q = head < p.nh, is_v = head >= p.nh + p.nkv;
    if (norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) ss += f[i] * f[i];
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (live && !is_v) {
        const float r = rsqrtf(ss / (float)p.hd + p.eps);
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = f[i] * r * (is_q ? wq[i] : wk[i]);
      }
    }
    if (!live) continue;
    if (!is_v && lane < f8) {
      const float2* cs = turn + tl * p.F + 8 * lane;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = f[i], b = f[8 + i];
        f[i] = a * cs[i].x - b * cs[i].y;
        f[8 + i] = b * cs[i].x + a * cs[i].y;
      }
    }
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = Elem<T>::pack(f[2 * i], f[2 * i + 1]);
    T* dst;
    if (is_q) {
      dst = static_cast<T*>(p.q_out) + ((int64_t)t * p.nh + head) * p.hd;
    } else {
      const int64_t slot = p.slots[t];
      if (slot < 0) continue;
      if (slot >= p.num_slots) {
        atomicExch(&g_paged_status, kErrBadPosition);
        continue;
      }
      const int64_t page = slot / p.page_size, row = slot - page * p.page_size;
      const int h = head - p.nh - (is_v ? p.nkv : 0);
      dst = static_cast<T*>(is_v ? p.v : p.k) + page * (is_v ? p.v_page : p.k_page) +
            ((int64_t)h * p.page_size + row) * p.hd;
    }
    *reinterpret_cast<uint4*>(dst + 8 * v0) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(dst + 8 * v1) = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// ---------------------------------------------------------------------------------------------------- attention
// One warp per new token and query head: the keys in blocks of 32, one a lane; running maximum and sum.
template <typename T, int HD>
__global__ void __launch_bounds__(128) attention_kernel(const PagedAttnParams p) {
  __shared__ float qs[4][HD];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + warp;
  if (item >= (int64_t)p.tokens * p.nh) return;
  const int t = (int)(item / p.nh), head = (int)(item % p.nh), kvh = head / (p.nh / p.nkv);
  int seq = 0;
  while (seq < p.seqs && p.cu_new[seq + 1] <= t) ++seq;
  if (seq == p.seqs) return;
  T* out = static_cast<T*>(p.out) + (int64_t)t * p.out_token + (int64_t)head * HD;
  int len = 0;
  if (t >= p.cu_new[seq]) len = min(p.seq_lens[seq], p.table_width * p.page_size) - (p.cu_new[seq + 1] - 1 - t);
  const T* q = static_cast<const T*>(p.q) + t * p.q_token + head * p.q_head;
  for (int d = lane; d < HD; d += 32) qs[warp][d] = Elem<T>::to_float(q[d]) * p.scale;
  __syncwarp();
  float m = -INFINITY, l = 0.f, o[HD / 32] = {};
  for (int j0 = 0; j0 < len; j0 += 32) {
    const int j = j0 + lane;
    int64_t at = -1;
    float sc = -INFINITY;
    if (j < len) {
      const int page = p.table[(int64_t)seq * p.table_stride + j / p.page_size];
      if (page < 0 || page >= p.num_pages) {
        atomicExch(&g_paged_status, kErrBadPosition);
      } else {
        at = ((int64_t)kvh * p.page_size + j % p.page_size) * HD;
        const T* k = static_cast<const T*>(p.k) + page * p.k_page + at;
        sc = 0.f;
        for (int d = 0; d < HD; ++d) sc += qs[warp][d] * Elem<T>::to_float(k[d]);
        at += page * p.v_page;
      }
    }
    float mx = sc;
#pragma unroll
    for (int o2 = 16; o2 > 0; o2 >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o2));
    mx = fmaxf(mx, m);
    const float base = mx == -INFINITY ? 0.f : mx;
    const float c = expf(m - base), pr = expf(sc - base);
    l = l * c + warp_sum(pr);
    m = mx;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) o[i] *= c;
    for (int jj = 0; jj < 32; ++jj) {
      const float pj = __shfl_sync(0xffffffffu, pr, jj);
      const int64_t aj = __shfl_sync(0xffffffffu, at, jj);
      if (aj < 0) continue;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) o[i] += pj * Elem<T>::to_float(static_cast<const T*>(p.v)[aj + lane + 32 * i]);
    }
  }
  for (int i = 0; i < HD / 32; ++i) out[lane + 32 * i] = Elem<T>::from_float(l > 0.f ? o[i] / l : 0.f);
}

template <typename Kern, typename P>
cudaError_t launch_paged(Kern kern, dim3 grid, dim3 block, size_t smem, bool pdl, cudaStream_t st, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <typename T>
cudaError_t append_t(const AppendParams& p, bool pdl, cudaStream_t st) {
  const int lanes = p.hd / 16, G = lanes <= 4 ? 4 : lanes <= 8 ? 8 : 16;
  const int per_token = (p.nh + 2 * p.nkv) * G;
  AppendParams a = p;
  a.tpb = per_token >= 256 ? 1 : 256 / per_token;
  const int threads = min(kAppendMaxThreads, (a.tpb * per_token + 31) / 32 * 32);
  auto kern = G == 4 ? append_kernel<T, 4> : G == 8 ? append_kernel<T, 8> : append_kernel<T, 16>;
  return launch_paged(kern, dim3((unsigned)((p.tokens + a.tpb - 1) / a.tpb)), dim3(threads),
                      (size_t)a.tpb * p.F * sizeof(float2), pdl, st, a);
}

template <typename T>
cudaError_t attention_t(const PagedAttnParams& p, bool pdl, cudaStream_t st) {
  const int64_t items = (int64_t)p.tokens * p.nh;
  return launch_paged(p.hd == 128 ? attention_kernel<T, 128> : attention_kernel<T, 64>,
                      dim3((unsigned)((items + 3) / 4)), dim3(128), 0, pdl, st, p);
}

}  // namespace

cudaError_t launch_paged_append(const void* qkv, int64_t ld, int64_t tokens, int nh, const void* q_norm,
                                const void* k_norm, float eps, const float* inv_freq, int rot, const int64_t* pos,
                                const int64_t* slots, const PagedCacheView& c, void* q_out, bool pdl, cudaStream_t st) {
  AppendParams p{qkv, ld, (int)tokens, nh, c.nkv, c.hd, rot / 2, q_norm, k_norm, eps, inv_freq, pos, slots, q_out,
                 c.k, c.v, c.k_page, c.v_page, c.num_pages * c.page_size, c.page_size, 1};
  return c.dtype == 0 ? append_t<__half>(p, pdl, st) : append_t<__nv_bfloat16>(p, pdl, st);
}

cudaError_t launch_paged_attention(const PagedAttnParams& p, bool pdl, cudaStream_t st) {
  return p.dtype == 0 ? attention_t<__half>(p, pdl, st) : attention_t<__nv_bfloat16>(p, pdl, st);
}

int paged_device_error() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_paged_status, sizeof(int));
  return v;
}

void paged_clear_device_error() {
  int z = 0;
  cudaMemcpyToSymbol(g_paged_status, &z, sizeof(int));
}

}  // namespace lb
