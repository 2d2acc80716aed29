// The paged KV cache: per-head norm + rotary rotation + append of a chunk of new tokens, and the attention of new
// tokens over the cache.
//
// Cache: K and V are [pages, nkv, page_size, hd], each page's block contiguous, pages a stride apart; a sequence's
// context lies in the pages its row of the page table lists, page_size tokens each.
#include <atomic>
#include <climits>

#include "lb_launch.h"
#include "lb_tc.cuh"
#include "lb_types.cuh"

namespace lb {

// status word of this file's kernels: a bounded wait that gave up, or a slot or page outside the cache
__device__ int g_paged_status;

namespace {

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
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t neg2(uint64_t a) {
  const float2 v = unpair(a);
  return pair(-v.x, -v.y);
}

// ------------------------------------------------------------------------------------------------------- append
// q and k heads: x <- x rsqrt(mean(x^2) + eps) w (where norm weights are given), then the pair (x_i, x_{i + F}),
// i < F, turned by the angle pos * f_i; the dimensions from 2F on are left as they are. v heads are copied. All in
// fp32, one rounding. Memory bound: each value is read once and written once.
//
// A group of G lanes takes one head of one token, 16 values a lane as two 16-byte vectors: lane j < F / 8 the vectors
// j and j + F / 8 (the two halves of eight pairs, so the rotation needs no exchange), the lanes after them two
// neighbouring vectors of the unrotated rest. A CTA holds up to four whole tokens. Once for all their heads it puts into
// shared memory the norm weights, each token's place in the cache and its cosines and sines -- the angle in fp64 as a
// multiple of pi (fp32 would lose 1e-3 of a turn at position 1e5) -- while the first values are already on their way;
// each group's next head is on its way while it works on one. 8192 tokens, 28 + 2 x 4 heads of 128: 32 us, 4.7 TB/s
// (75.6 with one token a CTA and the norm weights and angles fetched by every group).
constexpr int kAppendThreads = 256;    // five CTAs an SM (4 or 6: 34.6, 37.4 us; 288 threads, a token a pass, four: 33.8)
constexpr int kAppendTokens = 4;       // (2: 39 us, 8: 33.7)

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
  bool early;       // norm weights may be read before the wait on the previous kernel
};

template <typename T, int G>
__global__ void __launch_bounds__(kAppendThreads, 5) append_kernel(const AppendParams p) {
  extern __shared__ __align__(16) uint8_t append_smem[];   // norm weights [2][hd], cache offsets [tpb][2], cos, sin [tpb][F]
  float* weights = reinterpret_cast<float*>(append_smem);
  int64_t* place = reinterpret_cast<int64_t*>(weights + 2 * p.hd);
  float* cosines = reinterpret_cast<float*>(place + 2 * p.tpb);
  float* sines = cosines + p.tpb * p.F;
  pdl_launch_dependents();
  const int heads = p.nh + 2 * p.nkv, f8 = p.F / 8;
  const int t0 = blockIdx.x * p.tpb, nt = min(p.tpb, p.tokens - t0), units = nt * heads;
  const int lane = threadIdx.x % G, per = blockDim.x / G;
  const int v0 = lane < f8 ? lane : 2 * lane, v1 = lane < f8 ? lane + f8 : 2 * lane + 1;
  const bool on = lane < p.hd / 16, norm = p.q_norm != nullptr;
  if (!p.early) pdl_wait();
  if (norm)
    for (int i = threadIdx.x; i < 2 * p.hd; i += blockDim.x)
      weights[i] = Elem<T>::to_float(i < p.hd ? static_cast<const T*>(p.q_norm)[i] : static_cast<const T*>(p.k_norm)[i - p.hd]);
  if (p.early) pdl_wait();
  const T* qkv = static_cast<const T*>(p.qkv) + t0 * p.ld;
  T* q_out = static_cast<T*>(p.q_out) + (int64_t)t0 * p.nh * p.hd;
  int u = threadIdx.x / G, tl = u / heads, head = u - tl * heads;
  uint4 x[2] = {}, next[2] = {};   // lanes past the head dim hold zeros
  auto load = [&](uint4 (&d)[2], int unit, int tok, int h) {
    if (unit < units && on) {
      const T* src = qkv + tok * p.ld + h * p.hd;
      d[0] = ldg_cg_u128(src + 8 * v0);
      d[1] = ldg_cg_u128(src + 8 * v1);
    }
  };
  load(x, u, tl, head);
  for (int i = threadIdx.x; i < nt; i += blockDim.x) {
    const int64_t slot = p.slots[t0 + i];
    int64_t k = -1, v = -1;
    if (slot >= p.num_slots) {
      atomicExch(&g_paged_status, kErrBadPosition);
    } else if (slot >= 0) {
      const int64_t page = slot / p.page_size, row = (slot - page * p.page_size) * p.hd;
      k = page * p.k_page + row;
      v = page * p.v_page + row;
    }
    place[2 * i] = k;
    place[2 * i + 1] = v;
  }
  for (int i = threadIdx.x; i < nt * p.F; i += blockDim.x) {
    // angle / pi reduced to [-1, 1] in fp64
    const int tok = i / p.F;
    double a = (double)p.pos[t0 + tok] * (double)p.inv_freq[i - tok * p.F] * 0.31830988618379067154;
    a -= 2.0 * rint(a * 0.5);
    float sn, cs;
    sincospif((float)a, &sn, &cs);
    cosines[i] = cs;
    sines[i] = sn;
  }
  __syncthreads();
  for (int u0 = 0; u0 < units; u0 += per) {
    const bool live = u < units && on;
    const int tok = tl, h = head;
    u += per;
    head += per;
    while (head >= heads) head -= heads, ++tl;
    load(next, u, tl, head);
    uint64_t f[8];   // two values each: an fp32 pair takes one instruction, and those bound this kernel beside memory
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 a = Elem<T>::unpack(reinterpret_cast<const uint32_t*>(x)[i]);
      f[i] = pair(a.x, a.y);
    }
    const bool is_q = h < p.nh, is_v = h >= p.nh + p.nkv;
    if (norm) {
      uint64_t sq = mul2(f[0], f[0]);
#pragma unroll
      for (int i = 1; i < 8; ++i) sq = fma2(f[i], f[i], sq);
      const float2 both = unpair(sq);
      float ss = both.x + both.y;
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (live && !is_v) {
        const float r = rsqrtf(ss / (float)p.hd + p.eps);
        const ulonglong2* w0 = reinterpret_cast<const ulonglong2*>(weights + (is_q ? 0 : p.hd) + 8 * v0);
        const ulonglong2* w1 = reinterpret_cast<const ulonglong2*>(weights + (is_q ? 0 : p.hd) + 8 * v1);
        const uint64_t rr = pair(r, r);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const ulonglong2 a = w0[i], b = w1[i];
          f[2 * i] = mul2(mul2(f[2 * i], rr), a.x);
          f[2 * i + 1] = mul2(mul2(f[2 * i + 1], rr), a.y);
          f[4 + 2 * i] = mul2(mul2(f[4 + 2 * i], rr), b.x);
          f[5 + 2 * i] = mul2(mul2(f[5 + 2 * i], rr), b.y);
        }
      }
    }
    x[0] = next[0];
    x[1] = next[1];
    if (!live) continue;
    if (!is_v && lane < f8) {
      const ulonglong2* cs = reinterpret_cast<const ulonglong2*>(cosines + tok * p.F + 8 * lane);
      const ulonglong2* sn = reinterpret_cast<const ulonglong2*>(sines + tok * p.F + 8 * lane);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const ulonglong2 c = cs[i], d = sn[i];
        const uint64_t a0 = f[2 * i], a1 = f[2 * i + 1], b0 = f[4 + 2 * i], b1 = f[5 + 2 * i];
        f[2 * i] = fma2(a0, c.x, neg2(mul2(b0, d.x)));
        f[2 * i + 1] = fma2(a1, c.y, neg2(mul2(b1, d.y)));
        f[4 + 2 * i] = fma2(b0, c.x, mul2(a0, d.x));
        f[5 + 2 * i] = fma2(b1, c.y, mul2(a1, d.y));
      }
    }
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v = unpair(f[i]);
      w[i] = Elem<T>::pack(v.x, v.y);
    }
    T* dst;
    if (is_q) {
      dst = q_out + (tok * p.nh + h) * p.hd;
    } else {
      const int64_t at = place[2 * tok + is_v];
      if (at < 0) continue;
      dst = static_cast<T*>(is_v ? p.v : p.k) + at + (int64_t)(h - p.nh - (is_v ? p.nkv : 0)) * p.page_size * p.hd;
    }
    *reinterpret_cast<uint4*>(dst + 8 * v0) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(dst + 8 * v1) = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// ------------------------------------------------------------------------------------------- attention, few rows
// A decode step's attention (up to 64 query rows of a key head: new tokens x heads that share it). The rows of 16 at a
// time meet the whole context, so what counts is the stream of K and V; a cluster of C CTAs splits the context, each
// CTA's four warps take its blocks of 16 keys in turn.
//   * S^T = K Q^T and O^T = V^T P^T as mma.sync m16n8k16 with the keys, then the head dims, on the 16-row side: eight
//     query rows fill a whole n-tile (with the rows on the 16-row side half of each MMA and of O's registers would idle).
//   * K and V go from memory straight into fragments, 16 bytes a lane: the order of the dims inside a k-step of S is free
//     as long as Q's agrees, and V's pairs of keys are put together from two rows with byte permutes. No shared memory,
//     no barriers in the loop; a block of K is fetched while the one before is used, V while its scores are formed.
//   * the running maximum is moved only when a score exceeds it by 8 (in powers of two), so that the weights stay below
//     2^8 and most blocks cost one vote instead of shuffles and a rescale. Sums stay with their lane until the end.
//   * keys no row sees are masked by selection and their V rows replaced by zeros: cache rows past a context may hold NaN.
// The warps' (maximum, sum, O) are joined in shared memory, the CTAs' through distributed shared memory, in one fixed
// order. Few long contexts leave most SMs idle even so: then Z clusters share a context, and a second kernel joins their
// parts from a workspace.
// Bound by memory: 96 contexts of up to 8192 tokens, 28/4 heads of 128: 133 us for 742 MB (5.6 TB/s, uneven contexts
// included); 256 of 8192: 6.5 TB/s. One short context: 6.4 us, the chain of its loads. (Two blocks of keys a warp in
// flight: fewer CTAs an SM, slower.)
constexpr int kFewWarps = 4;
constexpr int kFewRows = 64;     // rows of a key head that go this way
constexpr int kFewCluster = 8;

template <typename T>
__device__ __forceinline__ void mma_rows(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if (Elem<T>::kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    mma16816(d, a0, a1, a2, a3, b0, b1);
}

// the transpose of an 8 x 8 matrix of 16-bit values held as one register a lane
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float ld_dsmem_f1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// A sequence's new tokens [t0, t0 + n) and context, kept inside the buffers whatever the arrays hold
struct SeqSpan {
  int t0, n, len;
};
__device__ __forceinline__ SeqSpan seq_span(const PagedAttnParams& p, int seq) {
  SeqSpan v;
  v.t0 = max(0, p.cu_new[seq]);
  v.n = min(p.cu_new[seq + 1], p.tokens) - v.t0;
  v.len = min(p.seq_lens[seq], p.table_width * p.page_size);
  return v;
}

template <typename T, int HD, int NT>   // NT: n-tiles of 8 query rows
__global__ void __launch_bounds__(32 * kFewWarps) attention_few_kernel(const PagedAttnParams p, int row_tiles, int C, int Z) {
  constexpr int kRows = 8 * NT, KI = HD / 32, VH = HD / 64;
  __shared__ __align__(16) float part[kFewWarps][kRows][HD + 4];
  __shared__ float part_m[kFewWarps][kRows], part_l[kFewWarps][kRows], cta_m[kRows], cta_l[kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = C > 1 ? (int)cluster_rank() : 0;
  int item = blockIdx.x / C;
  const int z = item % Z;
  item /= Z;
  const int work_row = item * kRows;   // this item's rows in the workspace
  const int rt = item % row_tiles;
  item /= row_tiles;
  const int kvh = item % p.nkv, seq = item / p.nkv, grp = p.nh / p.nkv;
  pdl_launch_dependents();
  pdl_wait();
  const int32_t* table = p.table + (int64_t)seq * p.table_stride;
  const int pages0 = lane < p.table_width ? table[lane] : 0;   // on its way together with the lengths
  const SeqSpan sp = seq_span(p, seq);
  const int rows = min(kRows, sp.n * grp - rt * kRows);   // of this tile (all the CTAs of a cluster agree)
  if (rows <= 0) return;
  const int row0 = rt * kRows;
  const int keys = min(sp.len, sp.len - sp.n + (row0 + rows - 1) / grp + 1);   // the last row's
  const int blocks = keys > 0 ? (keys + 15) / 16 : 0;
  const int share = z * C + rank, shares = Z * C;
  const int u0 = (int)((int64_t)blocks * share / shares), u1 = (int)((int64_t)blocks * (share + 1) / shares);

  // Q as the n-side operand, rows past the tile as zeros; the last key each of this lane's two rows per n-tile sees
  uint4 q[NT][KI];
  int last[NT][2];
  int first_masked = INT_MAX;   // blocks from this key on need the mask
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = 8 * nt + g;
#pragma unroll
    for (int i = 0; i < KI; ++i) q[nt][i] = make_uint4(0, 0, 0, 0);
    if (r < rows) {
      const int row = row0 + r;
      const T* src = static_cast<const T*>(p.q) + (int64_t)(sp.t0 + row / grp) * p.q_token + (int64_t)(kvh * grp + row % grp) * p.q_head;
#pragma unroll
      for (int i = 0; i < KI; ++i) q[nt][i] = ldg_cg_u128(src + 32 * i + 8 * t);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int rr = 8 * nt + 2 * t + e;
      last[nt][e] = rr < rows ? sp.len - sp.n + (row0 + rr) / grp : -1;
    }
  }
  first_masked = sp.len - sp.n + row0 / grp + 1;   // the first row's count of keys
  const float scale = p.scale * 1.44269504088896340736f;   // scores in powers of two

  const int per_page = p.page_size / 16;
  const T* kbase = static_cast<const T*>(p.k) + (int64_t)kvh * p.page_size * HD;
  const T* vbase = static_cast<const T*>(p.v) + (int64_t)kvh * p.page_size * HD;
  auto page_of = [&](int u, bool start) {   // start: the first lookups, which `pages0` may answer; -1: no such page
    const int at = u / per_page;
    int pg = 0;
    if (u < u1) pg = start && at < 32 ? __shfl_sync(0xffffffffu, pages0, at) : table[at];
    if (pg < 0 || pg >= p.num_pages) {
      atomicExch(&g_paged_status, kErrBadPosition);
      pg = -1;
    }
    return pg;
  };
  uint4 kf[KI][2], vf[VH][4];
  auto load_k = [&](int u, int pg) {
    const T* src = kbase + max(pg, 0) * p.k_page + (int64_t)(u % per_page) * 16 * HD + g * HD + 8 * t;
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      kf[i][0] = ldg_cg_u128(src + 32 * i);
      kf[i][1] = ldg_cg_u128(src + 8 * HD + 32 * i);
    }
  };
  auto load_v = [&](int u, int pg) {
    const T* src = vbase + max(pg, 0) * p.v_page + (int64_t)(u % per_page) * 16 * HD + 2 * t * HD + 8 * g;
#pragma unroll
    for (int h = 0; h < VH; ++h) {
      vf[h][0] = ldg_cg_u128(src + 64 * h);
      vf[h][1] = ldg_cg_u128(src + HD + 64 * h);
      vf[h][2] = ldg_cg_u128(src + 8 * HD + 64 * h);
      vf[h][3] = ldg_cg_u128(src + 9 * HD + 64 * h);
    }
  };

  float o[NT][VH][4][4] = {};
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.f;

  int u = u0 + warp;
  int page = page_of(u, true), page_next = page_of(u + kFewWarps, true);
  if (u < u1) load_k(u, page);
  for (; u < u1; u += kFewWarps) {
    load_v(u, page);
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        mma_rows<T>(s[nt], kf[i][0].x, kf[i][1].x, kf[i][0].y, kf[i][1].y, q[nt][i].x, q[nt][i].y);
        mma_rows<T>(s[nt], kf[i][0].z, kf[i][1].z, kf[i][0].w, kf[i][1].w, q[nt][i].z, q[nt][i].w);
      }
    }
    const int un = u + kFewWarps;
    // keys and values of a page outside the cache count as zeros: what was loaded in their place is dropped here, since
    // a branch around the loads costs every block (96 contexts of up to 8192: 134 -> 138 us)
    const bool absent = page < 0;
    if (absent) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
    }
    page = page_next;
    page_next = page_of(un + kFewWarps, false);
    if (un < u1) load_k(un, page);
    // scores in powers of two, unseen keys -inf; s[.][e] key g, row 2t + e; s[.][2 + e] key g + 8
    const bool masked = 16 * u + 16 > first_masked;
    bool move = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[nt][e] *= scale;
        if (masked && 16 * u + g + (e >= 2 ? 8 : 0) > last[nt][e & 1]) s[nt][e] = -INFINITY;
        move |= s[nt][e] > m[nt][e & 1] + 8.f;
      }
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(s[nt][e], s[nt][2 + e]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
          if (!(x > m[nt][e] + 8.f)) x = m[nt][e];   // (each row by its own scores, whatever stands beside it)
          const float c = x == m[nt][e] ? 1.f : exp2_fast(m[nt][e] - x);
          m[nt][e] = x;
          l[nt][e] *= c;
#pragma unroll
          for (int h = 0; h < VH; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[nt][h][i][e] *= c, o[nt][h][i][2 + e] *= c;
        }
    }
    uint32_t b[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float mm = m[nt][e & 1];
        w[e] = exp2_fast(s[nt][e] - (mm == -INFINITY ? 0.f : mm));
        l[nt][e & 1] += w[e];
      }
      b[nt][0] = transpose8(Elem<T>::pack(w[0], w[1]));
      b[nt][1] = transpose8(Elem<T>::pack(w[2], w[3]));
    }
    if (absent || 16 * u + 16 > keys) {   // V rows that no row of the tile sees
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (absent || 16 * u + 2 * t + (j & 1) + (j >= 2 ? 8 : 0) >= keys)
#pragma unroll
          for (int h = 0; h < VH; ++h) vf[h][j] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int h = 0; h < VH; ++h) {
      const uint32_t v[4][4] = {{vf[h][0].x, vf[h][0].y, vf[h][0].z, vf[h][0].w},
                                {vf[h][1].x, vf[h][1].y, vf[h][1].z, vf[h][1].w},
                                {vf[h][2].x, vf[h][2].y, vf[h][2].z, vf[h][2].w},
                                {vf[h][3].x, vf[h][3].y, vf[h][3].z, vf[h][3].w}};
#pragma unroll
      for (int i = 0; i < 4; ++i) {   // dims 64h + 8g + 2i (row g) and + 1 (row g + 8)
        const uint32_t a0 = __byte_perm(v[0][i], v[1][i], 0x5410), a1 = __byte_perm(v[0][i], v[1][i], 0x7632);
        const uint32_t a2 = __byte_perm(v[2][i], v[3][i], 0x5410), a3 = __byte_perm(v[2][i], v[3][i], 0x7632);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_rows<T>(o[nt][h][i], a0, a1, a2, a3, b[nt][0], b[nt][1]);
      }
    }
  }

  // join the warps: part[w][row][dim]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 8 * nt + 2 * t + e;
      float sum = l[nt][e];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (g == 0) part_m[warp][r] = m[nt][e], part_l[warp][r] = sum;
#pragma unroll
      for (int h = 0; h < VH; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float2*>(&part[warp][r][64 * h + 8 * g + 2 * i]) = make_float2(o[nt][h][i][e], o[nt][h][i][2 + e]);
    }
  __syncthreads();
  T* out = static_cast<T*>(p.out);
  auto store = [&](int r, int d, const float4& v, float sum) {
    const int row = row0 + r;
    const float c = sum != 0.f ? 1.f / sum : 0.f;
    *reinterpret_cast<uint2*>(out + (int64_t)(sp.t0 + row / grp) * p.out_token + (int64_t)(kvh * grp + row % grp) * HD + d) =
        make_uint2(Elem<T>::pack(v.x * c, v.y * c), Elem<T>::pack(v.z * c, v.w * c));
  };
  // four dims of a row a thread; the CTA's sum replaces warp 0's part
  for (int e = threadIdx.x; e < rows * (HD / 4); e += 32 * kFewWarps) {
    const int r = e / (HD / 4), d = e % (HD / 4) * 4;
    float mx = part_m[0][r];
#pragma unroll
    for (int w = 1; w < kFewWarps; ++w) mx = fmaxf(mx, part_m[w][r]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float c = part_m[w][r] == -INFINITY ? 0.f : exp2_fast(part_m[w][r] - mx);
      const float4 x = *reinterpret_cast<const float4*>(&part[w][r][d]);
      acc.x += c * x.x, acc.y += c * x.y, acc.z += c * x.z, acc.w += c * x.w;
      sum += c * part_l[w][r];
    }
    if (C == 1) {
      store(r, d, acc, sum);
    } else {
      *reinterpret_cast<float4*>(&part[0][r][d]) = acc;
      if (d == 0) cta_m[r] = mx, cta_l[r] = sum;
    }
  }
  if (C == 1) return;
  cluster_sync_all();
  for (int e = rank * 32 * kFewWarps + threadIdx.x; e < rows * (HD / 4); e += C * 32 * kFewWarps) {
    const int r = e / (HD / 4), d = e % (HD / 4) * 4;
    const uint32_t am = smem_addr(&cta_m[r]), al = smem_addr(&cta_l[r]), ao = smem_addr(&part[0][r][d]);
    float mk[kFewCluster], lk[kFewCluster];
    float4 x[kFewCluster];
#pragma unroll
    for (int k = 0; k < kFewCluster; ++k)   // (all of them under way together)
      if (k < C) {
        mk[k] = ld_dsmem_f1(mapa_shared(am, k));
        lk[k] = ld_dsmem_f1(mapa_shared(al, k));
        x[k] = ld_dsmem_f4(mapa_shared(ao, k));
      }
    float mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int k = 0; k < kFewCluster; ++k)
      if (k < C) mx = fmaxf(mx, mk[k]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < kFewCluster; ++k)
      if (k < C) {
        const float c = mk[k] == -INFINITY ? 0.f : exp2_fast(mk[k] - mx);
        acc.x += c * x[k].x, acc.y += c * x[k].y, acc.z += c * x[k].z, acc.w += c * x[k].w;
        sum += c * lk[k];
      }
    if (Z == 1) {
      store(r, d, acc, sum);
    } else {
      const int64_t at = (int64_t)(work_row + r) * Z + z;
      *reinterpret_cast<float4*>(p.work_o + at * HD + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(p.work_ml + 2 * at) = make_float2(mx, sum);
    }
  }
  cluster_sync_all();   // no CTA leaves while another still reads its part
}

// Joins the Z <= 32 parts of each row: work_o [item rows][Z][HD], work_ml [item rows][Z][2]. A CTA takes a row; its
// threads hold four dims of every 512 / HD-th part, all loads under way at once.
constexpr int kFewParts = 32;

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(128) attention_join_kernel(const PagedAttnParams p, int row_tiles, int Z) {
  constexpr int kRows = 8 * NT, kGroups = 512 / HD, kHeld = kFewParts / kGroups;
  __shared__ float4 sums[kGroups][HD / 4];
  __shared__ float weights[kGroups];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t work_row = blockIdx.x;
  const int group = threadIdx.x / (HD / 4), d = threadIdx.x % (HD / 4) * 4;
  float2 ml[kHeld];
  float4 x[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int k = group + i * kGroups;
    if (k < Z) {
      ml[i] = __ldcg(reinterpret_cast<const float2*>(p.work_ml + 2 * (work_row * Z + k)));
      x[i] = __ldcg(reinterpret_cast<const float4*>(p.work_o + (work_row * Z + k) * HD + d));
    }
  }
  float mx = (threadIdx.x & 31) < Z ? __ldcg(p.work_ml + 2 * (work_row * Z + (threadIdx.x & 31))) : -INFINITY;
  int item = (int)(work_row / kRows);
  const int row = item % row_tiles * kRows + (int)(work_row % kRows);
  item /= row_tiles;
  const int kvh = item % p.nkv, seq = item / p.nkv, grp = p.nh / p.nkv;
  const SeqSpan sp = seq_span(p, seq);
  if (row >= sp.n * grp) return;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (group + i * kGroups < Z) {
      const float c = ml[i].x == -INFINITY ? 0.f : exp2_fast(ml[i].x - mx);
      acc.x += c * x[i].x, acc.y += c * x[i].y, acc.z += c * x[i].z, acc.w += c * x[i].w;
      sum += c * ml[i].y;
    }
  sums[group][d / 4] = acc;
  if (d == 0) weights[group] = sum;
  __syncthreads();
  if (group) return;
  for (int k = 1; k < kGroups; ++k) {
    const float4 v = sums[k][d / 4];
    acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
    sum += weights[k];
  }
  const float c = sum != 0.f ? 1.f / sum : 0.f;
  T* dst = static_cast<T*>(p.out) + (int64_t)(sp.t0 + row / grp) * p.out_token + (int64_t)(kvh * grp + row % grp) * HD + d;
  *reinterpret_cast<uint2*>(dst) = make_uint2(Elem<T>::pack(acc.x * c, acc.y * c), Elem<T>::pack(acc.z * c, acc.w * c));
}

// ---------------------------------------------------------------------------------------- attention, chunks of tokens
// tcgen05 with two 128-row tiles of one key head's queries (new tokens x heads that share it) a CTA, over 128 keys at a
// time; one pass, running maximum and sum in registers, a query row per thread.
//   * loader warp: K and V tiles alternate in one ring of stages; a tile is put together from its pages, one tensor copy
//     per page (or part of a page: gcd(page size, 128) rows) and 128-byte half of a row, a lane each.
//   * MMA warp: S_t = Q_t K^T (K-major operands) into tensor memory, O_t += P_t V with P_t, the A operand, in tensor memory
//     over S_t's columns and V taken as it lies (MN-major B). PV of one tile and the next QK^T of the same tile are issued
//     together, so that while one tile's softmax runs the tensor core works for the other.
//     At hd 64 tensor memory holds a third tile of scores: QK^T then runs three row tiles ahead, and a softmax finds its
//     next scores there when it is done.
//   * two softmax warpgroups, one a tile: a thread reads its row's 128 scores at once, moves its running maximum only
//     when one exceeds it by 8 in powers of two (weights stay below 2^8; else O would be rescaled in tensor memory every
//     tile), writes the weights back as 16-bit pairs, and keeps their fp32 sum unrounded.
// Masks are applied by selection and only in tiles that reach past the first row's last key. V rows past the context may
// hold NaN, and 0 x NaN is NaN: a third warp zeroes them in shared memory before the last product.
// Weights are rounded to the 16-bit type for the second product, as tensor cores take it; scores, maxima, sums and O are
// fp32.
// Few tiles: a cluster of C CTAs splits the keys; each parks O, maxima and sums in its idle ring and all join their share
// of the rows through distributed shared memory, in one fixed order. (Pushing the parts to their owners instead: 33 us
// where this takes 29.)
// Bound by the softmax beside the MMAs: a step of 256 rows x 128 keys takes some 3100 clocks at hd 128, of which the MMAs
// need 2048, and 2700 at hd 64 (1024), with two warps a scheduler issuing 40 % of the time. 28/4 heads of 128: 4096 new
// tokens 117 us (1025 TFLOP/s), over 32768 1625 us (1110) in a first second of calls and 1760 (1025) once the power cap
// holds the clock; 14/2 of 64: 4096 over 16384 327 to 350 us (600 to 640; 370 with two score tiles). Neither MMAs issued by two warps (873 for 1072), nor two softmax threads a row (3 % more on long contexts, 7 %
// less on short ones) came out ahead.
__device__ __forceinline__ float max3(float a, float b, float c) {   // NaN if one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x of two values without the special-function unit: x = n + f with n the nearest integer (adding 1.5 * 2^23 leaves it
// in the low bits), 2^f on [-1/2, 1/2] by a polynomial of least relative error among those that are 1 at 0 (degree 3:
// 1.02e-4, under a bf16 weight's rounding; degree 4: 2.9e-6 for fp16), n added to the exponent. The 1 at 0 is for what
// lies below -127, an unseen key's -inf above all: there n = -127 and f = 0, and 127 taken from the exponent of 1 leaves
// the bits of exactly 0 (a least weight of 2^-126 would count beside a bf16 value of 2^127). Between -127 and -126 the
// result is off by at most 2^-126. (A product with 2^n instead of the addition: 3 % slower on long contexts.)
template <typename T>
__device__ __forceinline__ float2 exp2_poly(uint64_t x2) {
  float2 x = unpair(x2);
  x2 = pair(fmaxf(x.x, -127.f), fmaxf(x.y, -127.f));
  const uint64_t t = add2(x2, pair(12582912.f, 12582912.f));
  const uint64_t f = add2(x2, fma2(t, pair(-1.f, -1.f), pair(12582912.f, 12582912.f)));
  uint64_t r;
  if (Elem<T>::kBf16) {
    r = fma2(f, pair(0.05500905960798264f, 0.05500905960798264f), pair(0.24221096932888031f, 0.24221096932888031f));
    r = fma2(f, r, pair(0.6932829022407532f, 0.6932829022407532f));
    r = fma2(f, r, pair(1.f, 1.f));
  } else {
    r = fma2(f, pair(0.009582576341927052f, 0.009582576341927052f), pair(0.05590682849287987f, 0.05590682849287987f));
    r = fma2(f, r, pair(0.24024106562137604f, 0.24024106562137604f));
    r = fma2(f, r, pair(0.6931241154670715f, 0.6931241154670715f));
    r = fma2(f, r, pair(1.f, 1.f));
  }
  const float2 n = unpair(t), v = unpair(r);
  return make_float2(__int_as_float(__float_as_int(v.x) + (__float_as_int(n.x) << 23)),
                     __int_as_float(__float_as_int(v.y) + (__float_as_int(n.y) << 23)));
}

constexpr int kTileKeys = 128;
constexpr int kTileRows = 256;
constexpr int kChunkThreads = 12 * 32;   // loader, MMA, tail and an idle warp (a warpgroup), 8 softmax warps
constexpr int kChunkCluster = 8;

template <int HD>
struct ChunkSmem {
  static constexpr int kHalves = HD / 64;
  static constexpr int kPoly = HD == 128 ? 5 : 4;   // of 16 weights, those by polynomial (0, 3, 4, 5, 7, 8 tried)
  static constexpr int kStageBytes = kTileKeys * HD * 2;
  static constexpr int kDepth = 2;     // K and V tiles each in the ring (4 at hd 64: a longer loop, 6 % slower)
  static constexpr int kStages = 2 * kDepth;
  static constexpr int kScores = HD == 128 ? 2 : 3;   // score tiles beside two O in tensor memory
  static constexpr int kRound = HD == 128 ? 2 : 6;    // jobs until a row tile meets the same score tile again
  static constexpr int kQ = kTileRows * HD * 2;
  static constexpr int kBars = kQ + kStages * kStageBytes;                  // offset of the barriers
  static constexpr int kSlot = kBars + (2 * kStages + kRound + 2 * kScores + 8) * 8;
  static constexpr int kTotal = kSlot + 16 + 1024;                          // + alignment
};

struct ChunkParams {
  PagedAttnParams a;
  int piece;     // keys of one tensor copy
  int tiles;     // row tiles of the grid per key head
  int C;
};

// The grid's row tile x: its sequence (-1: past the last), the tile in it and the sequence's tokens. Tiles are counted
// longest first, so that the last CTAs to start are short: among each 32 sequences those of longer contexts come first,
// and a sequence's later rows, which see more keys, before its earlier ones. All lanes of a warp call it.
struct TilePlace {
  int seq, tile;
  SeqSpan span;
};
__device__ __forceinline__ TilePlace find_tile(const PagedAttnParams& p, int x, int grp) {
  const int lane = threadIdx.x & 31;
  for (int s0 = 0; s0 < p.seqs; s0 += 32) {
    int s = s0 + lane;
    SeqSpan sp = {0, 0, 0};
    if (s < p.seqs) sp = seq_span(p, s);
    if (p.seqs > 1) {   // lane i takes the sequence of rank i
      int rank = 0, from = lane;
      for (int i = 0; i < 32; ++i) {
        const int len = __shfl_sync(0xffffffffu, sp.len, i);
        rank += len > sp.len || (len == sp.len && i < lane);
      }
      for (int i = 0; i < 32; ++i) {
        const uint32_t who = __ballot_sync(0xffffffffu, rank == i);
        if (lane == i) from = __ffs(who) - 1;
      }
      s = s0 + from;
      sp = {__shfl_sync(0xffffffffu, sp.t0, from), __shfl_sync(0xffffffffu, sp.n, from), __shfl_sync(0xffffffffu, sp.len, from)};
    }
    const int mine = sp.n > 0 ? (int)(((int64_t)sp.n * grp + kTileRows - 1) / kTileRows) : 0;
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, sum > x);
    if (past) {
      const int at = __ffs(past) - 1;
      return {__shfl_sync(0xffffffffu, s, at), __shfl_sync(0xffffffffu, sum, at) - 1 - x,
              {__shfl_sync(0xffffffffu, sp.t0, at), __shfl_sync(0xffffffffu, sp.n, at), __shfl_sync(0xffffffffu, sp.len, at)}};
    }
    x -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return {-1, 0, {0, 0, 0}};
}

// a lane's pointer, as every lane sees it
template <typename T>
__device__ __forceinline__ T* shfl_ptr(T* v, int lane) {
  return reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(v), lane));
}

template <typename T, int HD>
__global__ void __launch_bounds__(kChunkThreads, 1)
    attention_chunk_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                           const ChunkParams cp) {
  using L = ChunkSmem<HD>;
  constexpr int kHalves = L::kHalves, St = L::kStages, B = L::kScores, R = L::kRound;
  constexpr uint32_t kO = 128 * B;   // tensor memory: B score tiles, two O
  constexpr uint32_t kHalfK = kTileKeys * 128, kHalfQ = 128 * 128;   // bytes of a 64-dim half of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint8_t* ring = smem + L::kQ;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* empty = full + St;
  uint64_t* q_ready = empty + St;
  uint64_t* s_full = q_ready + 1;
  uint64_t* p_ready = s_full + R;   // [part][score tile]
  uint64_t* o_done = p_ready + 2 * B;
  uint64_t* drain = o_done + 2;
  uint64_t* tail_go = drain + 1;
  uint64_t* v_tail = drain + 2;
  uint64_t* o_last = drain + 3;     // with three score tiles a row tile's last two products may both be to come
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + L::kSlot);
  float* row_m = reinterpret_cast<float*>(smem);   // [256] each, over Q, which no product reads any more by then
  float* row_l = row_m + kTileRows;
  const PagedAttnParams& p = cp.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int C = cp.C, rank = C > 1 ? (int)cluster_rank() : 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < St; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_ready, 8);
    mbar_init(drain, 1);
    mbar_init(tail_go, 1);
    mbar_init(v_tail, 1);
    for (int i = 0; i < R; ++i) mbar_init(&s_full[i], 1);
    for (int i = 0; i < 2 * B; ++i) mbar_init(&p_ready[i], 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&o_done[i], 1);
      mbar_init(&o_last[i], 1);
    }
    mbar_fence_init();
  }
  if (warp == 1) tc::alloc(slot, 512);   // all there is: it starts at column 0
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  constexpr uint32_t tmem = 0;
  pdl_launch_dependents();
  pdl_wait();

  const int grp = p.nh / p.nkv, item = blockIdx.x / C;
  const int kvh = item % p.nkv;
  const TilePlace at = find_tile(p, item / p.nkv, grp);
  const int seq = at.seq, row0 = at.tile * kTileRows;
  const SeqSpan sp = at.span;
  int rows = 0, keys = 0;
  if (seq >= 0) {
    rows = min(kTileRows, sp.n * grp - row0);
    keys = max(0, min(sp.len, sp.len - sp.n + (row0 + rows - 1) / grp + 1));   // the last row's
  }
  const int key_tiles = (keys + kTileKeys - 1) / kTileKeys;
  const int j0 = (int)((int64_t)key_tiles * rank / C), nt = (int)((int64_t)key_tiles * (rank + 1) / C) - j0;

  // 128 x 56 + 256 x 224 registers are the launch's 384 x 168: a softmax thread holds its row's 128 scores. (The
  // warpgroups' paths do not meet again before the end: what follows a meeting has the fewer registers.)
  if (warp < 4) {
    tc::regs_dec<56>();
    if (warp == 0) {
      if (seq >= 0 && nt > 0) {
        if (lane == 0) {
          tma_prefetch_map(&kmap);
          tma_prefetch_map(&vmap);
        }
        // lane -> (piece, half); table entries one tile ahead
        const int pieces = kTileKeys / cp.piece, piece = lane / kHalves, half = lane % kHalves;
        const bool mine = piece < pieces;
        const int32_t* table = p.table + (int64_t)seq * p.table_stride;
        const int per_page = p.page_size / cp.piece;
        const uint32_t dst0 = half * kHalfK + piece * cp.piece * 128;
        auto lookup = [&](int j, int& page, int& row) {   // this lane's piece of key tile j
          const int key = (j0 + j) * kTileKeys + piece * cp.piece;
          page = -1;
          if (mine && j < nt && key < keys) {
            const int idx = key / cp.piece, tp = idx / per_page;
            row = kvh * p.page_size + (idx - tp * per_page) * cp.piece;
            // past the cache: the tensor map's first page that is not there, of which the copy writes zeros
            const uint32_t listed = (uint32_t)table[tp], pages = (uint32_t)p.num_pages;
            page = (int)min(listed, pages);
            if (listed >= pages && half == 0) atomicExch(&g_paged_status, kErrBadPosition);
          }
        };
        int page, row = 0, page_next, row_next = 0;
        lookup(0, page, row);
        // whole pieces, a power of two of keys each
        const int last_keys = min(keys - (j0 + nt - 1) * kTileKeys, kTileKeys);
        const uint32_t last_bytes = (uint32_t)((last_keys + cp.piece - 1) & -cp.piece) * (128 * kHalves);
        int s = 0, phase = 0, filled = 0;
        bool ok = true;   // of this lane: nothing in the loop takes the whole warp, so that one that gave up can leave alone
        for (int j = 0; j < nt && ok; ++j) {
          lookup(j + 1, page_next, row_next);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            if (filled >= St) ok = wait_bounded(&empty[s], phase, &g_paged_status);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(&full[s], j + 1 < nt ? L::kStageBytes : last_bytes);
            if (page >= 0)
              tc::tma_load_3d(smem_addr(ring) + s * L::kStageBytes + dst0, kv ? &vmap : &kmap, 64 * half, row, page, &full[s]);
            ++filled;
            if (++s == St) s = 0, phase ^= filled > St;
          }
          page = page_next, row = row_next;
        }
        // no copy in flight past this point
        const int last = min(filled, St);
        for (int i = 0; i < last; ++i) {
          const int f = filled - last + i;
          wait_bounded(&full[f % St], (f / St) & 1, &g_paged_status);
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // One elected lane runs the whole loop (measured, eight MMAs with a wait and a commit: 570 clocks this way, 660 when the
      // warp loops and elects at each group, 840 under `if (lane == 0)`; they take 512). It shares its scheduler with two
      // softmax warps, so an instruction costs it ten clocks: the ring is unrolled and every address a constant offset.
      if (seq >= 0 && nt > 0 && tc::elect_one()) {
        constexpr uint32_t kType = Elem<T>::kBf16 ? (1u << 7) | (1u << 10) : 0u;
        constexpr uint32_t kQK = (1u << 4) | kType | ((kTileKeys >> 3) << 17) | ((128u >> 4) << 24);
        constexpr uint32_t kPV = (1u << 4) | kType | (1u << 16) | ((HD >> 3) << 17) | ((128u >> 4) << 24);   // B MN-major
        constexpr int D = L::kDepth;
        constexpr uint32_t kStep = L::kStageBytes >> 4;
        uint32_t kd = (uint32_t)tc::desc_sw128(smem_addr(ring), 16, 1024);
        uint32_t vd = (uint32_t)tc::desc_sw128(smem_addr(ring) + L::kStageBytes, kHalfK, 1024);
        uint32_t qd = (uint32_t)tc::desc_sw128(smem_addr(smem), 16, 1024);
        const uint32_t bars = smem_addr(full);
        constexpr uint32_t kEmpty = 8 * St, kQReady = 16 * St, kSFull = kQReady + 8, kPReady = kSFull + 8 * R, kODone = kPReady + 16 * B,
                           kDrain = kODone + 16, kTailGo = kDrain + 8, kVTail = kDrain + 16, kOLast = kDrain + 24;
        auto wait = [&](uint32_t off, uint32_t parity) { return wait_ready(bars + off, parity, &g_paged_status); };
        int b = 0;         // of the job at hand: its score tile, and the parity of that tile's uses
        uint32_t bp = 0;
        auto qk = [&](int b, int i, int t, int d) {   // the scores of a job i (mod R): row tile t with K stage d
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)
            tc::mma_f16_ss(tmem + 128 * b, qd + ((t * kHalves * kHalfQ + (k / 4) * kHalfQ + (k % 4) * 32) >> 4),
                           kd + 2 * d * kStep + (((k / 4) * kHalfK + (k % 4) * 32) >> 4), kQK, k > 0);
          tc::commit_at(bars + kSFull + 8 * i);
        };
        // tile j with V stage u, and the scores B jobs on, which take the score tile just used; false when a wait gave up
        auto step = [&](int j, int u, uint32_t ring_parity, bool first, bool more) {
          asm volatile("" : "+r"(kd), "+r"(vd), "+r"(qd));   // (or the compiler keeps every sum in a register of its own)
          if (!wait(8 * (2 * u + 1), ring_parity)) return false;
          if (!more && keys - (j0 + j) * kTileKeys < kTileKeys) {   // the third warp's turn
            mbar_arrive(tail_go);
            if (!wait(kVTail, 0)) return false;
          }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int at = B == 2 ? t : b;
#pragma unroll
            for (int part = 0; part < 2; ++part) {
              if (!wait(kPReady + 8 * (B * part + at), B == 2 ? u & 1 : bp)) return false;
              tc::fence_after();
#pragma unroll
              for (int k = part ? 6 : 0; k < (part ? 8 : 6); ++k)
                tc::mma_f16_ts(tmem + kO + HD * t, tmem + 128 * at + 8 * k, vd + 2 * u * kStep + ((k * 2048) >> 4), kPV,
                               !first || k > 0);
            }
            tc::commit_at(bars + kODone + 8 * t);
            if (B > 2 && !more) tc::commit_at(bars + kOLast + 8 * t);
            if (t == 1) tc::commit_at(bars + kEmpty + 8 * (2 * u + 1));
            const int tn = (t + B) & 1, un = u + (t + B) / 2;   // of job 2j + t + B
            if (j + (t + B) / 2 < nt) {
              if (tn == 0) {
                if (!wait(8 * (2 * (un % D)), un / D % 2 ? ring_parity ^ 1 : ring_parity)) return false;
                tc::fence_after();
              }
              qk(at, B == 2 ? t : bp ? b : b + B, tn, un % D);
              if (tn == 1) tc::commit_at(bars + kEmpty + 8 * (2 * (un % D)));
            }
            if (B > 2 && ++b == B) b = 0, bp ^= 1;
          }
          return true;
        };
        bool ok = wait(kQReady, 0) && wait(0, 0);
        tc::fence_after();
        if (ok) {
          qk(0, 0, 0, 0);
          qk(1, 1, 1, 0);
          tc::commit_at(bars + kEmpty);
          if (B > 2 && nt > 1) {
            ok = wait(16, 0);
            tc::fence_after();
            if (ok) qk(2, 2, 0, 1);
          }
        }
        uint32_t parity = 0;
        for (int j = 0; j < nt && ok; j += D, parity ^= 1) {
#pragma unroll
          for (int u = 0; u < D; ++u)
            if (ok && j + u < nt) ok = step(j + u, u, parity, j + u == 0, j + u + 1 < nt);
        }
        // no MMA in flight past this point
        tc::commit_at(bars + kDrain);
        wait(kDrain, 0);
      }
      __syncwarp();
    } else if (warp == 2) {
      // the V rows behind the context in the last tile, zeroed once the tile has arrived
      const int tail = keys - (j0 + nt - 1) * kTileKeys;
      if (seq >= 0 && nt > 0 && tail < kTileKeys) {
        const int fill = 2 * nt - 1;
        wait_bounded(tail_go, 0, &g_paged_status);
        uint8_t* tile = ring + (fill % St) * L::kStageBytes;
        for (int half = 0; half < kHalves; ++half)
          for (int i = lane; i < (kTileKeys - tail) * 8; i += 32)
            *reinterpret_cast<uint4*>(tile + half * kHalfK + tail * 128 + i * 16) = make_uint4(0, 0, 0, 0);
        tc::fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_tail);
      }
      __syncwarp();
    }
    if (C > 1) {
      cluster_sync_all();
      cluster_sync_all();
    }
  } else {
    tc::regs_inc<224>();
    const int t = (warp - 4) >> 2, quarter = warp & 3, r = 128 * t + 32 * quarter + lane, row = row0 + r;
    const uint32_t lane_base = tmem + ((uint32_t)(32 * quarter) << 16);
    const uint32_t to = lane_base + kO + HD * t;
    int job = t;                // modulo R
    uint32_t job_parity = 0;
    const bool on = r < rows;
    float m = -INFINITY, l = 0.f;
    const float scale = p.scale * 1.44269504088896340736f;
    const int last = on ? sp.len - sp.n + row / grp : -1;
    const int64_t token = sp.t0 + row / grp, head = (int64_t)kvh * grp + row % grp;
    uint8_t* stage = smem + t * kHalves * kHalfQ + 32 * quarter * 128;   // the warp's rows of Q, swizzled
    if (seq >= 0 && nt > 0) {
      // the warp's 32 rows, HD / 8 lanes a row at a time (a row a lane took three times as long)
      const T* mine = on ? static_cast<const T*>(p.q) + token * p.q_token + head * p.q_head : nullptr;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        const int rr = i * (256 / HD) + lane / (HD / 8), c = lane % (HD / 8);
        const T* src = shfl_ptr(mine, rr);
        const uint4 v = src ? ldg_cg_u128(src + 8 * c) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(stage + rr * 128 + (c / 8) * kHalfQ + (((c % 8) ^ (rr & 7)) << 4)) = v;
      }
      tc::fence_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
      const int first_last = sp.len - sp.n + row0 / grp;   // the CTA's first row's last key
      bool ok = true;   // of this lane: one that gave up waits no more, but stays with its warp's collective instructions
      for (int j = 0; j < nt; ++j) {
        const uint32_t at = B == 2 ? t : job < B ? job : job - B, ts = lane_base + 128 * at;
        if (ok) ok = wait_bounded(&s_full[B == 2 ? t : job], B == 2 ? j & 1 : job_parity, &g_paged_status);
        __syncwarp();
        tc::fence_after();
        uint32_t v[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tc::ld32(ts + 32 * c, v[c]);
        tc::wait_ld();
        const int k0 = (j0 + j) * kTileKeys;
        if (k0 + kTileKeys - 1 > first_last) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (k0 + 32 * c + i > last) v[c][i] = 0xFF800000u;   // -inf
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[c] = max3(__uint_as_float(v[c][0]), __uint_as_float(v[c][1]), __uint_as_float(v[c][2]));
#pragma unroll
          for (int i = 3; i < 31; i += 2) mx[c] = max3(mx[c], __uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1]));
          mx[c] = max3(mx[c], __uint_as_float(v[c][31]), __uint_as_float(v[c][31]));
        }
        const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * scale;
        // a score that is NaN or +inf makes the row NaN, as exp(inf - inf) would; the polynomial below would hide it
        if (!(top < INFINITY)) l = NAN;
        // (each row by its own scores alone, so that its result does not depend on the rows beside it)
        const bool move = top > m + 8.f && top < INFINITY;
        if (__any_sync(0xffffffffu, move)) {
          const float mn = move ? top : m;
          const float c = move ? exp2_fast(m - mn) : 1.f;
          m = mn;
          l *= c;
          if (j > 0) {   // the last product of this tile is complete before O is touched
            if (ok) ok = wait_bounded(&o_done[t], (j - 1) & 1, &g_paged_status);
            __syncwarp();
            tc::fence_after();
#pragma unroll
            for (int h = 0; h < HD / 32; ++h) {
              uint32_t o[32];
              tc::ld32(to + 32 * h, o);
              tc::wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * c);
              tc::st32(to + 32 * h, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.f : m;
        const uint64_t scale2 = pair(scale, scale), base2 = pair(-base, -base);
        uint64_t sum = pair(0.f, 0.f);
        // handed over in two parts: the products with the first 96 keys' V begin under the last weights
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t x = fma2(pair(__uint_as_float(v[c][2 * i]), __uint_as_float(v[c][2 * i + 1])), scale2, base2);
            float2 e;
            if ((i * L::kPoly) % 16 < L::kPoly) {
              e = exp2_poly<T>(x);
            } else {
              e = unpair(x);
              e.x = exp2_fast(e.x), e.y = exp2_fast(e.y);
            }
            sum = add2(sum, pair(e.x, e.y));
            w[i] = Elem<T>::pack(e.x, e.y);
          }
          tc::st16(ts + 16 * c, w);
          if (c >= 2) {
            tc::wait_st();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[B * (c - 2) + at]);
          }
        }
        const float2 both = unpair(sum);
        l += both.x + both.y;
        job += 2;
        if (job >= R) job -= R, job_parity ^= 1;
      }
      wait_bounded(B == 2 ? &o_done[t] : &o_last[t], B == 2 ? (nt - 1) & 1 : 0, &g_paged_status);
      __syncwarp();
      tc::fence_after();
    }
    if (C == 1) {
      if (seq >= 0) {
        // through the warp's rows of Q, which are done with, so that HD / 8 lanes store a row at a time
        const float c = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int h = 0; h < HD / 32; ++h) {
          uint32_t o[32];
          if (nt > 0) {
            tc::ld32(to + 32 * h, o);
            tc::wait_ld();
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = l != 0.f ? Elem<T>::pack(__uint_as_float(o[8 * i + 2 * e]) * c, __uint_as_float(o[8 * i + 2 * e + 1]) * c) : 0u;
            const int piece = 4 * h + i;
            *reinterpret_cast<uint4*>(stage + lane * 128 + (piece / 8) * kHalfQ + (((piece % 8) ^ (lane & 7)) << 4)) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
        T* mine = on ? static_cast<T*>(p.out) + token * p.out_token + head * HD : nullptr;
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
          const int rr = i * (256 / HD) + lane / (HD / 8), piece = lane % (HD / 8);
          const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * 128 + (piece / 8) * kHalfQ + (((piece % 8) ^ (rr & 7)) << 4));
          T* dst = shfl_ptr(mine, rr);
          if (dst) *reinterpret_cast<uint4*>(dst + 8 * piece) = v;
        }
      }
    } else {
      // the second tile's last product is the last to read the ring
      if (seq >= 0 && nt > 0) wait_bounded(B == 2 ? &o_done[1] : &o_last[1], B == 2 ? (nt - 1) & 1 : 0, &g_paged_status);
      __syncwarp();
      tc::fence_after();
      // parked at ring + row * HD * 4, 16-byte pieces permuted by the row so that eight lanes' stores take all banks
      row_m[r] = nt > 0 ? m : -INFINITY;
      row_l[r] = nt > 0 ? l : 0.f;
      if (seq >= 0 && nt > 0) {
#pragma unroll
        for (int h = 0; h < HD / 32; ++h) {
          uint32_t o[32];
          tc::ld32(to + 32 * h, o);
          tc::wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4*>(ring + r * HD * 4 + (((8 * h + i) ^ (r & 7)) << 4)) =
                make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
    }
    __syncwarp();
    if (C > 1) {
      cluster_sync_all();
      if (seq >= 0) {
        // a share of the rows a CTA, HD / 4 lanes a row
        constexpr int kLanes = HD / 4;
        const int c4 = (threadIdx.x - 128) % kLanes;
        constexpr int kPass = 256 / kLanes, kAtOnce = 2;   // rows a pass, and passes under way together
        for (int r0 = rank * kPass + (threadIdx.x - 128) / kLanes; r0 < rows; r0 += kAtOnce * C * kPass) {
          float mk[kAtOnce][kChunkCluster], lk[kAtOnce][kChunkCluster];
          float4 x[kAtOnce][kChunkCluster];
#pragma unroll
          for (int n = 0; n < kAtOnce; ++n) {
            const int r = min(r0 + n * C * kPass, kTileRows - 1);
            const uint32_t am = smem_addr(row_m + r), al = smem_addr(row_l + r);
            const uint32_t ao = smem_addr(ring) + r * HD * 4 + ((c4 ^ (r & 7)) << 4);
#pragma unroll
            for (int k = 0; k < kChunkCluster; ++k)
              if (k < C) {
                mk[n][k] = ld_dsmem_f1(mapa_shared(am, k));
                lk[n][k] = ld_dsmem_f1(mapa_shared(al, k));
                x[n][k] = ld_dsmem_f4(mapa_shared(ao, k));
              }
          }
#pragma unroll
          for (int n = 0; n < kAtOnce; ++n) {
            const int r = r0 + n * C * kPass, row = row0 + r;
            if (r >= rows) break;
            float mx = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < kChunkCluster; ++k)
              if (k < C) mx = fmaxf(mx, mk[n][k]);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < kChunkCluster; ++k)
              if (k < C && lk[n][k] != 0.f) {   // (a part without keys holds whatever its ring held)
                const float c = exp2_fast(mk[n][k] - mx);
                acc.x += c * x[n][k].x, acc.y += c * x[n][k].y, acc.z += c * x[n][k].z, acc.w += c * x[n][k].w;
                sum += c * lk[n][k];
              }
            const float c = sum != 0.f ? 1.f / sum : 0.f;
            T* dst = static_cast<T*>(p.out) + (int64_t)(sp.t0 + row / grp) * p.out_token + ((int64_t)kvh * grp + row % grp) * HD + 4 * c4;
            *reinterpret_cast<uint2*>(dst) = make_uint2(Elem<T>::pack(acc.x * c, acc.y * c), Elem<T>::pack(acc.z * c, acc.w * c));
          }
        }
      }
      cluster_sync_all();
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    tc::dealloc(tmem, 512);
  }
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
  // whole tokens a CTA: what fills 256 threads, and up to four where there are many
  a.tpb = max(256 / per_token, (int)min((int64_t)kAppendTokens, (int64_t)p.tokens / (4 * sm_count())));
  a.tpb = max(1, min(a.tpb, p.tokens));
  const int threads = min(kAppendThreads, (a.tpb * per_token + 31) / 32 * 32);
  auto kern = G == 4 ? append_kernel<T, 4> : G == 8 ? append_kernel<T, 8> : append_kernel<T, 16>;
  return launch_paged(kern, dim3((unsigned)((p.tokens + a.tpb - 1) / a.tpb)), dim3(threads),
                      (size_t)2 * p.hd * sizeof(float) + a.tpb * 16 + (size_t)a.tpb * p.F * sizeof(float2), pdl, st, a);
}

// CTAs of the few-rows kernel that can be resident at once in clusters of C, on the current device
template <int HD, int NT>
int few_resident(int C) {
  static std::atomic<int> known[64][kFewCluster + 1];   // + 1; 0: not asked yet
  int dev = 0;
  cudaGetDevice(&dev);
  int v = known[dev & 63][C].load(std::memory_order_relaxed);
  if (v == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(C);
    cfg.blockDim = dim3(32 * kFewWarps);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, attention_few_kernel<__half, HD, NT>, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 2 * sm_count() / C;
    }
    v = n * C + 1;
    known[dev & 63][C].store(v, std::memory_order_relaxed);
  }
  return v - 1;
}

// How few rows are laid out: tiles of 8 or 16 rows, clusters of C CTAs, Z clusters a context -- the choice whose estimated
// time is least, in microseconds as measured: 4 to start and end a CTA; a block of keys and warp 1.5 (hd 64: 0.95), by one
// in a thousand CTAs more, or what memory takes for all CTAs' blocks together; 1 to join a cluster, 4 for the second
// kernel; CTAs past those resident at once come in further rounds. Where a warp has more than 36 blocks each costs 1
// more, since contexts differ and the longest ends last (36 and 1 fit contexts spread evenly up to 8192, the last line below;
// they are not derived). (C = 1, 2, 3, 4, 6: 32 contexts of 4096, 28/4 heads of 128 100, 60, 47,
// 66, 53 us; 64 of 4096 110, 124, 92, 104, 104; 100 of 3000, 16/2 heads 79, 53, 68, 58, 64; 96 of up to 8192, 28/4 heads
// 196, 146, 135, 131, 134.)
struct FewPlan {
  int nt, row_tiles, C, Z;
  int64_t items;
};
FewPlan few_plan(int64_t rows, int64_t seqs, int nkv, int hd, int64_t max_len) {
  FewPlan f;
  f.nt = rows <= 8 ? 1 : 2;
  f.row_tiles = (int)((rows + 8 * f.nt - 1) / (8 * f.nt));
  f.items = seqs * nkv * f.row_tiles;
  const int64_t blocks = (max_len + 15) / 16;
  double least = 1e30;
  f.C = f.Z = 1;
  for (int C = 1; C <= kFewCluster; ++C) {
    const double resident = hd == 128 ? (f.nt == 1 ? few_resident<128, 1>(C) : few_resident<128, 2>(C))
                                      : (f.nt == 1 ? few_resident<64, 1>(C) : few_resident<64, 2>(C));
    for (int Z = 1; Z <= (C == kFewCluster ? kFewParts : 1); ++Z) {
      if (C * Z > 1 && blocks < 2 * C * Z) break;
      const int64_t turns = (blocks + C * Z * kFewWarps - 1) / (C * Z * kFewWarps);
      const double ctas = (double)(f.items * C * Z), rounds = floor(ctas / resident), rest = ctas - rounds * resident;
      auto round = [&](double n) {
        return 4 + (C > 1) + turns * max((hd == 128 ? 1.5 : 0.95) + 0.001 * n, n * kFewWarps * 16 * hd * 4 / 6.2e6);
      };
      double t = rounds * round(resident) + (rest > 0 ? round(rest) : 0) + (Z > 1 ? 4 : 0);
      if (turns > 36) t += turns;
      if (t < least) least = t, f.C = C, f.Z = Z;
    }
  }
  return f;
}

template <typename T, int HD, int NT>
cudaError_t few_t(PagedAttnParams p, const FewPlan& f, bool pdl, cudaStream_t st) {
  const int64_t rows = f.items * 8 * NT;
  p.work_ml = static_cast<float*>(p.workspace);
  p.work_o = p.work_ml + (2 * rows * f.Z + 3) / 4 * 4;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(f.items * f.Z * f.C));
  cfg.blockDim = dim3(32 * kFewWarps);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  if (pdl) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  const int joined_attrs = cfg.numAttrs;
  if (f.C > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = f.C;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = attr;
  cudaError_t e = cudaLaunchKernelEx(&cfg, attention_few_kernel<T, HD, NT>, (const PagedAttnParams)p, f.row_tiles, f.C, f.Z);
  if (e != cudaSuccess || f.Z == 1) return e;
  cfg.gridDim = dim3((unsigned)rows);
  cfg.blockDim = dim3(128);
  cfg.numAttrs = joined_attrs;
  return cudaLaunchKernelEx(&cfg, attention_join_kernel<T, HD, NT>, (const PagedAttnParams)p, f.row_tiles, f.Z);
}

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// Clusters of C CTAs of the chunk kernel that can be resident at once
template <int HD>
int chunk_resident(int C) {
  static std::atomic<int> known[64][kChunkCluster + 1];
  int dev = 0;
  cudaGetDevice(&dev);
  int v = known[dev & 63][C].load(std::memory_order_relaxed);
  if (v == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(C);
    cfg.blockDim = dim3(kChunkThreads);
    cfg.dynamicSmemBytes = ChunkSmem<HD>::kTotal;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, attention_chunk_kernel<__half, HD>, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = max(1, (sm_count() - 16) / C);
    }
    v = n;
    known[dev & 63][C].store(v, std::memory_order_relaxed);
  }
  return v;
}

template <typename T, int HD>
cudaError_t chunk_t(const PagedAttnParams& p, bool pdl, cudaStream_t st) {
  using L = ChunkSmem<HD>;
  auto kern = attention_chunk_kernel<T, HD>;
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (!(done.load(std::memory_order_relaxed) & bit)) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(attention_chunk_kernel<__half, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal);
    if (e != cudaSuccess) return e;
    done.fetch_or(bit, std::memory_order_relaxed);
  }
  ChunkParams cp;
  cp.a = p;
  cp.piece = gcd(p.page_size, kTileKeys);
  const int64_t grp = p.nh / p.nkv;
  // every sequence's last tile may be partial
  cp.tiles = (int)min(p.seqs * ((p.max_new * grp + kTileRows - 1) / kTileRows), (p.tokens * grp + kTileRows - 1) / kTileRows + p.seqs);
  const int64_t items = (int64_t)cp.tiles * p.nkv, key_tiles = (p.max_len + kTileKeys - 1) / kTileKeys;
  // The cluster that costs least: rounds of CTAs times their key tiles (1.4 us each, measured) and 6 us to start and end,
  // 6 more to join a cluster (C = 1, 2, 3, 4: 300 tokens over 4096, 28/4 heads of 128 61, 44, 35, 49 us; 1000 over 1000,
  // 16/2 heads 21, 24, 33, 32; 500 over 2000, 14/2 heads of 64 29, 23, 20, 17)
  double least = 1e30;
  cp.C = 1;
  for (int C = 1; C <= kChunkCluster && (C == 1 || key_tiles >= 2 * C); ++C) {
    const int64_t resident = C == 1 ? sm_count() : chunk_resident<HD>(C), rounds = (items + resident - 1) / resident;
    const double t = (double)rounds * (6 + (C > 1 ? 6 : 0) + 1.4 * (double)((key_tiles + C - 1) / C));
    if (t < least) least = t, cp.C = C;
  }
  CUtensorMap kmap, vmap;
  const CUtensorMapDataType type = Elem<T>::kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t extent[3] = {(uint64_t)HD, (uint64_t)p.nkv * p.page_size, (uint64_t)p.num_pages};
  const uint32_t box[3] = {64, (uint32_t)cp.piece, 1};
  const uint64_t ks[2] = {(uint64_t)HD * 2, (uint64_t)p.k_page * 2}, vs[2] = {(uint64_t)HD * 2, (uint64_t)p.v_page * 2};
  if (!encode_tensor_map_3d(&kmap, type, p.k, extent, ks, box, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_tensor_map_3d(&vmap, type, p.v, extent, vs, box, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(items * cp.C));
  cfg.blockDim = dim3(kChunkThreads);
  cfg.dynamicSmemBytes = L::kTotal;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  if (pdl) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cp.C > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cp.C;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kern, kmap, vmap, cp);
}

template <typename T>
cudaError_t attention_t(const PagedAttnParams& p, bool pdl, cudaStream_t st) {
  const int64_t most_rows = (int64_t)p.max_new * (p.nh / p.nkv);
  if (most_rows <= kFewRows) {
    const FewPlan f = few_plan(most_rows, p.seqs, p.nkv, p.hd, p.max_len);
    return p.hd == 128 ? (f.nt == 1 ? few_t<T, 128, 1>(p, f, pdl, st) : few_t<T, 128, 2>(p, f, pdl, st))
                       : (f.nt == 1 ? few_t<T, 64, 1>(p, f, pdl, st) : few_t<T, 64, 2>(p, f, pdl, st));
  }
  return p.hd == 128 ? chunk_t<T, 128>(p, pdl, st) : chunk_t<T, 64>(p, pdl, st);
}

}  // namespace

cudaError_t launch_paged_append(const void* qkv, int64_t ld, int64_t tokens, int nh, const void* q_norm,
                                const void* k_norm, float eps, const float* inv_freq, int rot, const int64_t* pos,
                                const int64_t* slots, const PagedCacheView& c, void* q_out, bool early, bool pdl,
                                cudaStream_t st) {
  AppendParams p{qkv, ld, (int)tokens, nh, c.nkv, c.hd, rot / 2, q_norm, k_norm, eps, inv_freq, pos, slots, q_out,
                 c.k, c.v, c.k_page, c.v_page, c.num_pages * c.page_size, c.page_size, 1, early};
  return c.dtype == 0 ? append_t<__half>(p, pdl, st) : append_t<__nv_bfloat16>(p, pdl, st);
}

size_t paged_attention_workspace(int64_t seqs, int nh, int nkv, int hd, int64_t max_new, int64_t max_len) {
  const int64_t rows = max_new * (nh / nkv);
  if (rows > kFewRows) return 0;
  const FewPlan f = few_plan(rows, seqs, nkv, hd, max_len);
  if (f.Z == 1) return 0;
  return (size_t)((2 * f.items * 8 * f.nt * f.Z + 3) / 4 * 4 + f.items * 8 * f.nt * f.Z * hd) * sizeof(float);
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
