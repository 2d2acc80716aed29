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
#include "lb_tma.cuh"
#include "lb_types.cuh"

namespace lb {

// status word of this file's kernels (a bounded wait that gave up); read by w8_device_error()
__device__ int g_w8_status;

namespace {

// ------------------------------------------------------------------------------------------- quantize rows
// One CTA per row: |x| maximum over the row, then the quantized bytes. Memory bound: reads 2 K (4 K for fp32) and
// writes K bytes a row; the row's second reading comes from L1 / L2.
constexpr int kQThreads = 256;

// q = rint(x * r), 127 / amax computed on amax * up so that the quotient of a row of subnormals stays finite
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
__device__ __forceinline__ int quant1(float x, const RowScale& v) {
  return max(-127, min(127, __float2int_rn(x * v.up * v.r)));
}

// the larger of |x| so far and |x|, keeping a NaN
__device__ __forceinline__ float amax_nan(float a, float x) {
  x = fabsf(x);
  return (x > a || x != x) ? x : a;
}

template <typename T>
__global__ void __launch_bounds__(kQThreads)
    quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, int ldq, float* __restrict__ s,
                         int K) {
  __shared__ float red[kQThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  float a = 0.f;
  for (int k = threadIdx.x; k < K; k += kQThreads) a = amax_nan(a, Elem<T>::to_float(xr[k]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = amax_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
  __syncthreads();
  a = red[0];
#pragma unroll
  for (int w = 1; w < kQThreads / 32; ++w) a = amax_nan(a, red[w]);
  const RowScale v = row_scale(a);
  if (threadIdx.x == 0) s[row] = v.s;
  for (int k = threadIdx.x; k < ldq; k += kQThreads)
    q[row * ldq + k] = k < K ? (int8_t)quant1(Elem<T>::to_float(xr[k]), v) : (int8_t)0;
}

// ------------------------------------------------------------------------------------------- the product
constexpr int kTile = 64;

template <typename T>
__global__ void __launch_bounds__(256)
    w8_gemm_kernel(const int8_t* __restrict__ q, const float* __restrict__ s, const int8_t* __restrict__ w,
                   const float* __restrict__ t, const T* __restrict__ bias, T* __restrict__ y, int M, int N, int ld) {
  __shared__ int qs[kTile][9], ws[kTile][9];   // 32 bytes of k per row, padded
  pdl_launch_dependents();
  pdl_wait();
  const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < ld; k0 += 32) {
    for (int i = threadIdx.x; i < kTile * 8; i += 256) {
      const int r = i >> 3, c = i & 7, k = k0 + 4 * c;
      qs[r][c] = m0 + r < M && k < ld ? *reinterpret_cast<const int*>(q + (int64_t)(m0 + r) * ld + k) : 0;
      ws[r][c] = n0 + r < N && k < ld ? *reinterpret_cast<const int*>(w + (int64_t)(n0 + r) * ld + k) : 0;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(qs[ty + 16 * i][c], ws[tx + 16 * j][c], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m < M && n < N)
        y[(int64_t)m * N + n] = Elem<T>::from_float(__int2float_rn(acc[i][j]) * s[m] * t[n] +
                                                    (bias ? Elem<T>::to_float(bias[n]) : 0.f));
    }
}

template <typename Kern, typename... Args>
cudaError_t launch_w8(Kern kern, dim3 grid, dim3 block, size_t smem, bool pdl, cudaStream_t st, Args... args) {
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
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <typename T>
cudaError_t linear_t(const W8Params& p, bool pdl, cudaStream_t st) {
  int8_t* q = static_cast<int8_t*>(p.workspace);
  float* s = reinterpret_cast<float*>(q + p.M * p.ldw);
  cudaError_t e = launch_w8(quantize_rows_kernel<T>, dim3((unsigned)p.M), dim3(kQThreads), 0, pdl, st,
                            static_cast<const T*>(p.x), p.ldx, q, (int)p.ldw, s, (int)p.K);
  if (e != cudaSuccess) return e;
  return launch_w8(w8_gemm_kernel<T>, dim3((unsigned)((p.N + 63) / 64), (unsigned)((p.M + 63) / 64)), dim3(256), 0,
                   pdl, st, (const int8_t*)q, (const float*)s, static_cast<const int8_t*>(p.w), p.w_scales,
                   static_cast<const T*>(p.bias), static_cast<T*>(p.y), (int)p.M, (int)p.N, (int)p.ldw);
}

}  // namespace

size_t w8_workspace_bytes(int64_t M, int64_t N, int64_t ldw) { return (size_t)M * (size_t)ldw + (size_t)M * 4; }

cudaError_t launch_w8_quantize_rows(const void* x, int dtype, int64_t ldx, int8_t* q, int64_t ldq, float* s, int64_t M,
                                    int64_t K, bool pdl, cudaStream_t st) {
  const dim3 grid((unsigned)M), block(kQThreads);
  switch (dtype) {
    case 0:
      return launch_w8(quantize_rows_kernel<__half>, grid, block, 0, pdl, st, static_cast<const __half*>(x), ldx, q,
                       (int)ldq, s, (int)K);
    case 1:
      return launch_w8(quantize_rows_kernel<__nv_bfloat16>, grid, block, 0, pdl, st,
                       static_cast<const __nv_bfloat16*>(x), ldx, q, (int)ldq, s, (int)K);
    default:
      return launch_w8(quantize_rows_kernel<float>, grid, block, 0, pdl, st, static_cast<const float*>(x), ldx, q,
                       (int)ldq, s, (int)K);
  }
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
