// The paged KV cache: per-head norm + rotary rotation + append of a chunk of new tokens, and the attention of new
// tokens over the cache.
//
// Cache: K and V are [pages, nkv, page_size, hd], each page's block contiguous, pages a stride apart; a sequence's
// context lies in the pages its row of the page table lists, page_size tokens each.
#include <atomic>
#include <climits>

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
// order.
constexpr int kFewWarps = 4;
constexpr int kFewRows = 64;   // rows of a key head that go this way

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
__global__ void __launch_bounds__(32 * kFewWarps) attention_few_kernel(const PagedAttnParams p, int row_tiles, int C) {
  constexpr int kRows = 8 * NT, KI = HD / 32, VH = HD / 64;
  __shared__ float part[kFewWarps][kRows][HD + 4];
  __shared__ float part_m[kFewWarps][kRows], part_l[kFewWarps][kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = C > 1 ? (int)cluster_rank() : 0;
  int item = blockIdx.x / C;
  const int rt = item % row_tiles;
  item /= row_tiles;
  const int kvh = item % p.nkv, seq = item / p.nkv, grp = p.nh / p.nkv;
  pdl_launch_dependents();
  pdl_wait();
  const SeqSpan sp = seq_span(p, seq);
  const int rows = min(kRows, sp.n * grp - rt * kRows);   // of this tile (all the CTAs of a cluster agree)
  if (rows <= 0) return;
  const int row0 = rt * kRows;
  const int keys = min(sp.len, sp.len - sp.n + (row0 + rows - 1) / grp + 1);   // the last row's
  const int blocks = keys > 0 ? (keys + 15) / 16 : 0;
  const int u0 = (int)((int64_t)blocks * rank / C), u1 = (int)((int64_t)blocks * (rank + 1) / C);

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

  const int32_t* table = p.table + (int64_t)seq * p.table_stride;
  const int per_page = p.page_size / 16;
  const T* kbase = static_cast<const T*>(p.k) + (int64_t)kvh * p.page_size * HD;
  const T* vbase = static_cast<const T*>(p.v) + (int64_t)kvh * p.page_size * HD;
  auto page_of = [&](int u) {
    int pg = u < u1 ? table[u / per_page] : 0;
    if (pg < 0 || pg >= p.num_pages) {
      atomicExch(&g_paged_status, kErrBadPosition);
      pg = 0;
    }
    return pg;
  };
  uint4 kf[KI][2], vf[VH][4];
  auto load_k = [&](int u, int pg) {
    const T* src = kbase + pg * p.k_page + (int64_t)(u % per_page) * 16 * HD + g * HD + 8 * t;
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      kf[i][0] = ldg_cg_u128(src + 32 * i);
      kf[i][1] = ldg_cg_u128(src + 8 * HD + 32 * i);
    }
  };
  auto load_v = [&](int u, int pg) {
    const T* src = vbase + pg * p.v_page + (int64_t)(u % per_page) * 16 * HD + 2 * t * HD + 8 * g;
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
  int page = page_of(u), page_next = page_of(u + kFewWarps);
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
    page = page_next;
    page_next = page_of(un + kFewWarps);
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
          x = fmaxf(x, m[nt][e]);
          const float c = x == -INFINITY ? 1.f : exp2_fast(m[nt][e] - x);
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
    if (16 * u + 16 > keys) {   // V rows that no row of the tile sees
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (16 * u + 2 * t + (j & 1) + (j >= 2 ? 8 : 0) >= keys)
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
  auto store = [&](int r, int d, float v) {
    const int row = row0 + r;
    out[(int64_t)(sp.t0 + row / grp) * p.out_token + (int64_t)(kvh * grp + row % grp) * HD + d] = Elem<T>::from_float(v);
  };
  // a thread takes the dims d, d + 128 mod HD of a row; the CTA's sum replaces warp 0's part
  for (int e = threadIdx.x; e < rows * HD; e += 32 * kFewWarps) {
    const int r = e / HD, d = e % HD;
    float mx = part_m[0][r];
#pragma unroll
    for (int w = 1; w < kFewWarps; ++w) mx = fmaxf(mx, part_m[w][r]);
    float acc = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float c = part_m[w][r] == -INFINITY ? 0.f : exp2_fast(part_m[w][r] - mx);
      acc += c * part[w][r][d];
      sum += c * part_l[w][r];
    }
    if (C == 1)
      store(r, d, sum > 0.f ? acc / sum : 0.f);
    else
      part[0][r][d] = acc;
  }
  if (C == 1) return;
  __shared__ float cta_m[kRows], cta_l[kRows];
  if (threadIdx.x < rows) {
    const int r = threadIdx.x;
    float mx = part_m[0][r], sum = 0.f;
    for (int w = 1; w < kFewWarps; ++w) mx = fmaxf(mx, part_m[w][r]);
    for (int w = 0; w < kFewWarps; ++w) sum += part_m[w][r] == -INFINITY ? 0.f : exp2_fast(part_m[w][r] - mx) * part_l[w][r];
    cta_m[r] = mx;
    cta_l[r] = sum;
  }
  cluster_sync_all();
  for (int e = rank * 32 * kFewWarps + threadIdx.x; e < rows * HD; e += C * 32 * kFewWarps) {
    const int r = e / HD, d = e % HD;
    const uint32_t am = smem_addr(&cta_m[r]), al = smem_addr(&cta_l[r]), ao = smem_addr(&part[0][r][d]);
    float mx = -INFINITY, acc = 0.f, sum = 0.f;
#pragma unroll 4
    for (int k = 0; k < C; ++k) mx = fmaxf(mx, ld_dsmem_f1(mapa_shared(am, k)));
#pragma unroll 4
    for (int k = 0; k < C; ++k) {
      const float mk = ld_dsmem_f1(mapa_shared(am, k));
      const float c = mk == -INFINITY ? 0.f : exp2_fast(mk - mx);
      acc += c * ld_dsmem_f1(mapa_shared(ao, k));
      sum += c * ld_dsmem_f1(mapa_shared(al, k));
    }
    store(r, d, sum > 0.f ? acc / sum : 0.f);
  }
  cluster_sync_all();   // no CTA leaves while another still reads its part
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

template <typename T, int HD, int NT>
cudaError_t few_t(const PagedAttnParams& p, bool pdl, cudaStream_t st) {
  const int row_tiles = (int)(((int64_t)p.max_new * (p.nh / p.nkv) + 8 * NT - 1) / (8 * NT));
  const int64_t items = (int64_t)p.seqs * p.nkv * row_tiles;
  const int sms = sm_count(), blocks = (p.max_len + 15) / 16;
  int C = 1;
  while (C < 8 && items * C < 6 * sms && blocks > C * 2 * kFewWarps) C *= 2;
  auto kern = attention_few_kernel<T, HD, NT>;
  if (items * C < sms && blocks > 32 * kFewWarps) {   // few long contexts: a cluster beyond the portable size
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (!(done.load(std::memory_order_relaxed) & bit)) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return e;
      done.fetch_or(bit, std::memory_order_relaxed);
    }
    C = 16;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(items * C));
  cfg.blockDim = dim3(32 * kFewWarps);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  if (pdl) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (C > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = C;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kern, p, row_tiles, C);
}

template <typename T>
cudaError_t attention_t(const PagedAttnParams& p, bool pdl, cudaStream_t st) {
  const int64_t most_rows = (int64_t)p.max_new * (p.nh / p.nkv);
  if (most_rows <= kFewRows)
    return p.hd == 128 ? (most_rows <= 8 ? few_t<T, 128, 1>(p, pdl, st) : few_t<T, 128, 2>(p, pdl, st))
                       : (most_rows <= 8 ? few_t<T, 64, 1>(p, pdl, st) : few_t<T, 64, 2>(p, pdl, st));
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
