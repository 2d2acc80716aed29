// A step of drafted tokens around the attention: the plan of a call (page tables, slots, positions and tree masks from the
// request lengths), the acceptance of the drafts, and the move of the accepted tokens' rows in the paged cache.
#include <atomic>

#include "lb_launch.h"
#include "lb_tma.cuh"
#include "lb_types.cuh"

namespace lb {

// status word of this file's kernels: a row outside the cache
__device__ int g_draft_status;

namespace {

__device__ __forceinline__ int ldg_cg_i32(const int32_t* p) { return (int)ldg_cg_u32(reinterpret_cast<const uint32_t*>(p)); }
__device__ __forceinline__ int64_t ldg_cg_i64(const int64_t* p) { return __ldcg(reinterpret_cast<const long long*>(p)); }

// --------------------------------------------------------------------------------------------------------- plan
// A few bytes of arithmetic a token behind two prefix sums over the sequences: latency. 16 trees of up to 31 tokens 6.1 us, 48
// prompts of up to 2048 tokens 6.4 (11.3 with eight CTAs at most, which met on the way), in a graph. Every CTA sums all sequences by
// itself (they are read once more from L2, which costs less than handing the sums over), then writes its share, without
// meeting the others. Where outputs lie over the inputs the grid is one cluster of up to eight CTAs, which meet once, before
// the first of them writes.
// With pages to give out, sequence s takes free_pages[count - 1 - first_s - j] as its page held_s + j, first_s being the
// sum of what the sequences before it need: the pages a loop over the sequences would pop from a stack. A token's slot on a
// new page is taken from that list too, not from the table that another CTA is writing.
constexpr int kPlanThreads = 1024;
constexpr int kPlanCluster = 8;
constexpr int kPlanStage = 2048;     // tokens of a tree round; their parents, and those before them in the first one's sequence, are staged

struct PlanSmem {   // per sequence: first token, tokens cached, pages taken before it, pages held (-1: refused)
  int *cu, *len, *first, *held;
};

// exclusive prefix sum over the CTA's threads; `total` receives the sum
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* warps, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
  int64_t sum = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += o;
  }
  __syncthreads();   // (the last call's sums are read)
  if (lane == 31) warps[warp] = sum;
  __syncthreads();
  int64_t before = lane < n ? warps[lane] : 0, all = before;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, all, d);
    if (lane >= d) all += o;
  }
  *total = __shfl_sync(0xffffffffu, all, 31);
  return __shfl_sync(0xffffffffu, all - before, warp) + sum - v;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p, int C, bool meet) {
  extern __shared__ int plan_smem[];
  __shared__ int64_t warps[32];
  __shared__ unsigned long long taken;   // pages of the sequences that are served
  const PlanSmem m{plan_smem, plan_smem + p.seqs + 1, plan_smem + 2 * p.seqs + 1, plan_smem + 3 * p.seqs + 1};
  int* stage = plan_smem + 4 * p.seqs + 1;
  const int rank = blockIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  const bool whole = p.parents && C == 1 && p.tokens <= kPlanStage;   // all parents are staged, on their way under the sums
  if (whole)
    for (int t = threadIdx.x; t < p.tokens; t += blockDim.x) stage[t] = ldg_cg_i32(p.parents + t);
  if (threadIdx.x == 0) taken = 0;
  const int64_t room = (int64_t)p.table_width * p.page_size;
  const int64_t count = p.free_count ? max(0, min(ldg_cg_i32(p.free_count), p.num_free)) : 0;
  int64_t tokens = 0, pages = 0;   // of the sequences so far
  for (int s0 = 0; s0 < p.seqs; s0 += blockDim.x) {
    const int s = s0 + threadIdx.x;
    const bool on = s < p.seqs;
    int64_t n = 0, len = 0;
    int held = 0;
    if (on) {
      n = min((int64_t)max(0, ldg_cg_i32(p.new_lens + s)), (int64_t)p.tokens + 1);
      len = max(0, ldg_cg_i32(p.seq_lens + s));
      if (p.held) held = max(0, ldg_cg_i32(p.held + s));
    }
    int64_t sum;
    const int64_t at = tokens + block_scan(n, warps, &sum);
    tokens += sum;
    bool served = (n == 0 || at + n <= p.tokens) && len + n <= room && (!p.parents || n <= 32 * p.words);
    const int64_t need = p.held && served ? max((int64_t)0, (len + n + p.page_size - 1) / p.page_size - held) : 0;
    const int64_t first = pages + block_scan(need, warps, &sum);
    pages += sum;
    served = served && (need == 0 || first + need <= count);
    if (served && need > 0) atomicMax(&taken, (unsigned long long)(first + need));   // those that are served come first
    if (on) {
      m.cu[s] = (int)min(at, (int64_t)p.tokens);
      m.len[s] = (int)len;
      m.first[s] = (int)min(first, count);
      m.held[s] = served ? held : -1 - held;
    }
  }
  if (threadIdx.x == 0) m.cu[p.seqs] = (int)min(tokens, (int64_t)p.tokens);
  if (meet)
    cluster_sync_all();   // every CTA has read what the outputs lie over
  else
    __syncthreads();

  // the sequences' share: a warp each
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, all_warps = (blockDim.x >> 5) * C;
  for (int s = rank * (blockDim.x >> 5) + warp; s < p.seqs; s += all_warps) {
    const int n = m.cu[s + 1] - m.cu[s], len = m.len[s], kept = m.held[s], held = kept < 0 ? -1 - kept : kept;
    const int need = p.held && kept >= 0 ? max(0, (int)(((int64_t)len + n + p.page_size - 1) / p.page_size) - held) : 0;
    for (int j = lane; j < need; j += 32)
      p.table[(int64_t)s * p.table_stride + held + j] = ldg_cg_i32(p.free_pages + count - 1 - m.first[s] - j);
    if (lane == 0) {
      p.cu_out[s] = m.cu[s];
      p.lens_out[s] = kept < 0 ? 0 : len + n;
      if (p.held) p.held_out[s] = held + need;
    }
  }
  if (rank == 0 && threadIdx.x == 0) {
    p.cu_out[p.seqs] = m.cu[p.seqs];
    if (p.free_count) p.free_count_out[0] = (int)(count - (int64_t)taken);
  }

  // a token's sequence: the last that starts at or before it and has tokens
  auto find = [&](int t) {
    int lo = 0, hi = p.seqs;   // cu[lo] <= t < cu[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (m.cu[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
  };
  auto place = [&](int t, int s, int depth) {
    const int i = t - m.cu[s], kept = m.held[s];
    const int64_t key = (int64_t)m.len[s] + i;
    int64_t slot = -1;
    if (kept >= 0) {
      const int pg = (int)((uint32_t)key / (uint32_t)p.page_size);   // below room, which fits 31 bits
      const bool taken_now = p.held && pg >= kept;
      const int page = ldg_cg_i32(taken_now ? p.free_pages + count - 1 - m.first[s] - (pg - kept)
                                            : p.table + (int64_t)s * p.table_stride + pg);
      slot = page < 0 ? -1 : (int64_t)page * p.page_size + (key - (int64_t)pg * p.page_size);
    }
    p.slots[t] = slot;
    p.positions[t] = (int64_t)m.len[s] + depth;
  };
  const int end = m.cu[p.seqs];
  if (!p.parents) {
    for (int t = rank * blockDim.x + threadIdx.x; t < p.tokens; t += blockDim.x * C) {
      if (t < end) {
        const int s = find(t);
        place(t, s, t - m.cu[s]);
      } else {
        p.slots[t] = -1;
        p.positions[t] = 0;
      }
    }
    return;
  }
  // G lanes a token, a word of its mask each; all of them walk up the tree
  int G = 1;
  while (G < p.words) G <<= 1;
  const int share = (p.tokens + C - 1) / C, t1 = min(p.tokens, (rank + 1) * share);
  for (int t0 = rank * share; t0 < t1; t0 += kPlanStage) {
    const int last = min(t1, t0 + kPlanStage);
    const int from = whole ? 0 : t0 < end ? max(m.cu[find(t0)], t0 - kMaxTree) : t0;   // a tree's parents may lie that far before
    if (!whole) {
      __syncthreads();
      for (int t = from + threadIdx.x; t < last; t += blockDim.x) stage[t - from] = ldg_cg_i32(p.parents + t);
      __syncthreads();
    }
    for (int u = threadIdx.x; u < (last - t0) * G; u += blockDim.x) {
      const int t = t0 + u / G, w = u % G;
      uint32_t bits = 0;
      if (t < end) {
        const int s = find(t), c = m.cu[s];
        int depth = 0;
        for (int i = t - c;;) {
          if (i >> 5 == w) bits |= 1u << (i & 31);
          const int at = c + i - from;
          const int up = at >= 0 ? stage[at] : -1;
          if (up < 0 || up >= i) break;   // no earlier token: a root
          i = up;
          ++depth;
        }
        if (w == 0) place(t, s, depth);
      } else if (w == 0) {
        p.slots[t] = -1;
        p.positions[t] = 0;
      }
      if (w < p.words) p.mask[(int64_t)t * p.words + w] = bits;
    }
  }
}

// ------------------------------------------------------------------------------------------------------- verify
// First each row's argmax, `splits` CTAs a row: bound by the logits' way from memory, so the loop takes only the maximum
// of kArgVecs 16-byte vectors a thread (packed, NaN above all) and remembers the first such group that exceeded what was
// there; the place inside the group is looked up once, by the threads whose maximum is the CTA's. 990 rows of 152064 bf16 values
// 52.6 us with the walk behind it, 5.75 TB/s, 88 % of a copy's rate; 8 rows of 151936 6.0 (two launches, the second released while the first runs).
constexpr int kArgThreads = 256;
constexpr int kArgVecs = 4;

// order-preserving bits of a value, NaN above all, -0 as +0; 0 is below every value
__device__ __forceinline__ uint32_t order_bits(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename T>
struct ArgVec {   // 16 bytes of a row
  static constexpr int kValues = 8;
  uint4 v;
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    if (Elem<T>::kBf16)
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ uint32_t most() const { return max2(max2(v.x, v.y), max2(v.z, v.w)); }
  static __device__ __forceinline__ uint32_t order(uint32_t packed) {
    const float2 f = Elem<T>::unpack(packed);
    return max(order_bits(f.x), order_bits(f.y));
  }
  static __device__ __forceinline__ uint32_t value(const T* p) {
    return order_bits(Elem<T>::unpack((uint32_t)ldg_cg_u16(p)).x);
  }
};
template <>
struct ArgVec<float> {
  static constexpr int kValues = 4;
  uint4 v;
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
    return __float_as_uint(r);
  }
  __device__ __forceinline__ uint32_t most() const { return max2(max2(v.x, v.y), max2(v.z, v.w)); }
  static __device__ __forceinline__ uint32_t order(uint32_t bits) { return order_bits(__uint_as_float(bits)); }
  static __device__ __forceinline__ uint32_t value(const float* p) {
    return order_bits(__uint_as_float(ldg_cg_u32(reinterpret_cast<const uint32_t*>(p))));
  }
};

template <typename T>
__global__ void __launch_bounds__(kArgThreads) argmax_kernel(const VerifyParams p, int splits) {
  using V = ArgVec<T>;
  constexpr int E = V::kValues;
  __shared__ uint32_t best_warp[kArgThreads / 32];
  __shared__ uint32_t best_at;
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x / splits, split = blockIdx.x - row * splits;
  if (row >= ldg_cg_i32(p.cu_new + p.seqs)) return;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.ld;
  const int head = min(p.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15u)) % 16 / sizeof(T)));   // values before the first whole vector
  const int vecs = (p.vocab - head) / E, v0 = (int)((int64_t)vecs * split / splits), v1 = (int)((int64_t)vecs * (split + 1) / splits);
  const T* xv = x + head;
  uint32_t best = 0;
  int at = 0;   // the first value of the group that holds it; groups are E values from `at` on, each kArgThreads vectors apart
  auto meet = [&](uint32_t o, int where) {
    if (o > best) best = o, at = where;
  };
  if (threadIdx.x == 0) best_at = 0xFFFFFFFFu;
  if (split == 0 && (int)threadIdx.x < head) meet(V::value(x + threadIdx.x), (int)threadIdx.x);
  for (int v = v0 + threadIdx.x; v < v1; v += kArgThreads * kArgVecs) {
    V g[kArgVecs];
#pragma unroll
    for (int i = 0; i < kArgVecs; ++i) {   // (past the end the first vector once more)
      const int w = v + i * kArgThreads < v1 ? v + i * kArgThreads : v;
      g[i].v = ldg_cg_u128(xv + (int64_t)w * E);
    }
    uint32_t o = g[0].most();
#pragma unroll
    for (int i = 1; i < kArgVecs; ++i) o = V::max2(o, g[i].most());
    meet(V::order(o), head + v * E);
  }
  const int tail = head + vecs * E + threadIdx.x;
  if (split == splits - 1 && tail < p.vocab) meet(V::value(x + tail), tail);
  uint32_t most = __reduce_max_sync(0xffffffffu, best);
  if ((threadIdx.x & 31) == 0) best_warp[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kArgThreads / 32; ++w) most = max(most, best_warp[w]);
  if (best == most && most != 0) {
    uint32_t found = 0xFFFFFFFFu;
    if (at < head || at >= head + vecs * E) {
      found = (uint32_t)at;
    } else {
      const int v = (at - head) / E;
#pragma unroll 1
      for (int i = 0; i < kArgVecs && found == 0xFFFFFFFFu; ++i) {
        const int w = v + i * kArgThreads;
        if (w < v1)
          for (int e = E - 1; e >= 0; --e)
            if (V::value(xv + (int64_t)w * E + e) == most) found = (uint32_t)(head + w * E + e);
      }
    }
    atomicMin(&best_at, found);
  }
  __syncthreads();
  // the larger value first, then the lower index
  if (threadIdx.x == 0) p.parts[(int64_t)row * splits + split] = (uint64_t)most << 32 | (uint32_t)~best_at;
}

// A CTA a sequence: its rows' targets from the parts, then one warp walks down the tree, 32 tokens at a time looked over for
// the next child. Latency.
constexpr int kWalkThreads = 128;

__global__ void __launch_bounds__(kWalkThreads) walk_kernel(const VerifyParams p, int splits) {
  __shared__ int64_t token[kMaxTree], target[kMaxTree];
  __shared__ int parent[kMaxTree];
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.x, t0 = max(0, ldg_cg_i32(p.cu_new + s));
  const int all = min(ldg_cg_i32(p.cu_new + s + 1), p.tokens) - t0, n = max(0, min(all, p.max_new));
  const bool served = n > 0 && (!p.seq_lens || ldg_cg_i32(p.seq_lens + s) >= all);   // (a refused one's rows have targets, but no path)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < n; i += kWalkThreads) {
    token[i] = ldg_cg_i64(p.drafted + t0 + i);
    parent[i] = ldg_cg_i32(p.parents + t0 + i);
  }
  // as many lanes a row as it has parts, up to a warp
  int G = 1;
  while (G < splits && G < 32) G <<= 1;
  const int sub = lane & (G - 1), groups = kWalkThreads / G;
  for (int i0 = 0; i0 < n; i0 += groups) {
    const int i = i0 + (warp * 32 + lane) / G;
    unsigned long long best = 0;
    if (i < n)
      for (int k = sub; k < splits; k += G) best = max(best, (unsigned long long)__ldcg(p.parts + (int64_t)(t0 + i) * splits + k));
    for (int d = G >> 1; d > 0; d >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, d));
    if (sub == 0 && i < n) {
      target[i] = (int64_t)(uint32_t)~(uint32_t)best;
      p.targets[t0 + i] = target[i];
    }
  }
  __syncthreads();
  if (warp) return;
  int cur = 0, length = served ? 1 : 0;
  int32_t* path = p.path + (int64_t)s * p.max_path;
  if (lane == 0) path[0] = served ? 0 : -1;
  while (length > 0 && length < p.max_path) {
    const int64_t want = target[cur];
    int child = -1;
    for (int c0 = cur + 1; c0 < n && child < 0; c0 += 32) {
      const int c = c0 + lane;
      const uint32_t hit = __ballot_sync(0xffffffffu, c < n && parent[c] == cur && token[c] == want);
      if (hit) child = c0 + __ffs(hit) - 1;
    }
    if (child < 0) break;
    cur = child;
    if (lane == 0) path[length] = cur;
    ++length;
  }
  for (int d = max(1, length) + lane; d < p.max_path; d += 32) path[d] = -1;
  if (lane == 0) {
    p.accepted[s] = length;
    p.next[s] = served ? target[cur] : -1;
  }
}

// ------------------------------------------------------------------------------------------------------ compact
// Row ctx + path[d] of each layer's K and V moves to ctx + d. A path rises, so a source lies at or behind its destination and
// behind every destination before it: a thread that takes one 16-byte column of a head through the whole path, eight rows
// loaded before the first of them is stored, overwrites nothing that is still to be read. A CTA works for one sequence; its
// first warps look up the rows once. One sequence is latency -- lengths and path, table, rows, one after another: 25 tokens in 36
// layers 2.6 us in a graph. A batch is at no bound: 64 trees in 28 layers 7.2 us, where the 12.6 MB read and written need 1.9; its
// 1792 CTAs each look the same up again for at most seven rows a thread.
constexpr int kMoveThreads = 128;    // (64 trees in 28 layers: 7.2 us; 256: 8.3, 64: 7.3)
constexpr int kMoveBatch = 8;

__global__ void __launch_bounds__(kMoveThreads) compact_kernel(const __grid_constant__ CompactParams p) {
  __shared__ int64_t src[kMoveThreads], dst[kMoveThreads];   // page << 32 | row; src < 0: the row stays where it is
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.y;
  const int32_t* path = p.path + (int64_t)s * p.max_path;
  int from = (int)threadIdx.x < p.max_path ? ldg_cg_i32(path + threadIdx.x) : 0;   // on its way together with the lengths
  const int n = max(0, ldg_cg_i32(p.cu_new + s + 1) - ldg_cg_i32(p.cu_new + s));
  const int len = ldg_cg_i32(p.seq_lens + s), start = len - n, length = min(ldg_cg_i32(p.accepted + s), min(p.max_path, n));
  if (len == 0 || start < 0) {   // a sequence that the plan refused (it may have no rows), or one that is empty: nothing to move
    if (!p.keep && blockIdx.x == 0 && threadIdx.x == 0) p.lens_out[s] = 0;
    return;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.lens_out[s] = start + max(0, length);
  const int lanes = p.hd / 8, items = 2 * p.layers * p.nkv, per = kMoveThreads / lanes;
  const int item = blockIdx.x * per + threadIdx.x / lanes, col = threadIdx.x % lanes * 8;
  const bool on = item < items && (int)threadIdx.x < per * lanes;
  const int kv = item & 1, layer = (item >> 1) / p.nkv, head = (item >> 1) % p.nkv;
  uint8_t* base = nullptr;
  int64_t page_stride = 0;
  if (on) {
    base = static_cast<uint8_t*>(kv ? p.v[layer] : p.k[layer]);
    page_stride = 2 * (kv ? p.v_page : p.k_page);
    base += 2 * ((int64_t)head * p.page_size * p.hd + col);
  }
  const int32_t* table = p.table + (int64_t)s * p.table_stride;
  for (int d0 = 0; d0 < length; d0 += kMoveThreads) {
    __syncthreads();
    const int d = d0 + threadIdx.x;
    if (d < length) {
      if (d0 > 0) from = ldg_cg_i32(path + d);
      int64_t place[2] = {-1, -1};
      bool ok = from >= d && from < n;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t key = (uint32_t)start + (uint32_t)(e ? d : from), pg = key / (uint32_t)p.page_size;
        const int page = ok && pg < (uint32_t)p.table_width ? ldg_cg_i32(table + pg) : -1;
        if (page < 0 || page >= p.num_pages) ok = false;
        place[e] = (int64_t)page << 32 | (key - pg * (uint32_t)p.page_size);
      }
      if (!ok) atomicExch(&g_draft_status, kErrBadPosition);
      src[threadIdx.x] = ok && from != d ? place[0] : -1;
      dst[threadIdx.x] = place[1];
    }
    __syncthreads();
    const int count = min(kMoveThreads, length - d0);
    auto at = [&](int64_t place) { return base + (place >> 32) * page_stride + (place & 0xFFFFFFFF) * (2 * p.hd); };
    if (on)
      for (int i0 = 0; i0 < count; i0 += kMoveBatch) {
        uint4 v[kMoveBatch];
#pragma unroll
        for (int i = 0; i < kMoveBatch; ++i)
          if (i0 + i < count && src[i0 + i] >= 0) v[i] = ldg_cg_u128(at(src[i0 + i]));
#pragma unroll
        for (int i = 0; i < kMoveBatch; ++i)
          if (i0 + i < count && src[i0 + i] >= 0) *reinterpret_cast<uint4*>(at(dst[i0 + i])) = v[i];
      }
  }
}

template <typename Kern, typename... Args>
cudaError_t launch_draft(Kern kern, dim3 grid, int threads, size_t smem, int cluster, bool pdl, cudaStream_t st, const Args&... args) {
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

// Two CTAs an SM where rows are few, with 4096 values each at least; three CTAs a row or so where they are many, so that the last
// round is short (990 rows of 152064: 57.9 us with one, 52.6 with three; 250 rows of 151936: 13.5 with two, 21.5 with fourteen)
int verify_splits(int64_t tokens, int64_t vocab) {
  const int64_t sms = sm_count(), few = min((2 * sms + tokens - 1) / tokens, vocab / 4096), many = min((16 * sms + tokens - 1) / tokens, vocab / 49152);
  return (int)max((int64_t)1, max(few, many));
}

}  // namespace

cudaError_t launch_plan(const PlanParams& p, bool pdl, cudaStream_t st) {
  auto over = [](const void* out, int64_t n, const void* in, int64_t k) {
    const auto a = reinterpret_cast<uintptr_t>(out), b = reinterpret_cast<uintptr_t>(in);
    return out && in && a < b + 4 * k && b < a + 4 * n;
  };
  bool meet = false;
  const void* ins[3] = {p.seq_lens, p.new_lens, p.held};
  for (const void* in : ins)
    meet |= over(p.lens_out, p.seqs, in, p.seqs) || over(p.held_out, p.seqs, in, p.seqs) || over(p.cu_out, p.seqs + 1, in, p.seqs) ||
            over(p.free_count_out, 1, in, p.seqs);
  meet |= over(p.free_count_out, 1, p.free_count, 1) || over(p.lens_out, p.seqs, p.free_count, 1) || over(p.held_out, p.seqs, p.free_count, 1);
  // one small CTA where that holds the work, else one for each 1024 threads' worth, to all SMs
  const int64_t work = (int64_t)p.tokens * (p.parents ? p.words : 1);
  int threads = work <= 512 && p.seqs <= 256 ? 256 : kPlanThreads, C = (int)max((int64_t)1, min((work + kPlanThreads - 1) / kPlanThreads, (int64_t)sm_count()));
  if (meet) C = work <= 2 * kPlanThreads ? 1 : work <= 8 * kPlanThreads ? 4 : kPlanCluster;
  meet = meet && C > 1;
  const size_t smem = (size_t)(4 * p.seqs + 1 + (p.parents ? kPlanStage + kMaxTree : 0)) * sizeof(int);
  if (smem > 48 * 1024) {   // once per device, what the largest call needs: a call's own size would take from another's under way
    static std::atomic<uint64_t> done{0};
    constexpr int kMost = (4 * kMaxPlanSeqs + 1 + kPlanStage + kMaxTree) * (int)sizeof(int);
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (!(done.load(std::memory_order_relaxed) & bit)) {
      const cudaError_t e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
      if (e != cudaSuccess) return e;
      done.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  return launch_draft(plan_kernel, dim3(C), threads, smem, meet ? C : 1, pdl, st, p, C, meet);
}

size_t verify_workspace_bytes(int64_t tokens, int64_t vocab) { return (size_t)tokens * verify_splits(tokens, vocab) * sizeof(uint64_t); }

cudaError_t launch_verify(const VerifyParams& p, bool pdl, cudaStream_t st) {
  const int splits = verify_splits(p.tokens, p.vocab);
  const dim3 grid((unsigned)(p.tokens * splits));
  const cudaError_t e =
      p.dtype == 0   ? launch_draft(argmax_kernel<__half>, grid, kArgThreads, 0, 1, pdl, st, p, splits)
      : p.dtype == 1 ? launch_draft(argmax_kernel<__nv_bfloat16>, grid, kArgThreads, 0, 1, pdl, st, p, splits)
                     : launch_draft(argmax_kernel<float>, grid, kArgThreads, 0, 1, pdl, st, p, splits);
  return e == cudaSuccess ? launch_draft(walk_kernel, dim3(p.seqs), kWalkThreads, 0, 1, pdl, st, p, splits) : e;
}

cudaError_t launch_compact(const CompactParams& p, bool pdl, cudaStream_t st) {
  const int per = kMoveThreads / (p.hd / 8), items = 2 * p.layers * p.nkv;
  return launch_draft(compact_kernel, dim3((items + per - 1) / per, p.seqs), kMoveThreads, 0, 1, pdl, st, p);
}

int draft_device_error() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_draft_status, sizeof(int));
  return v;
}

void draft_clear_device_error() {
  int z = 0;
  cudaMemcpyToSymbol(g_draft_status, &z, sizeof(int));
}

}  // namespace lb
