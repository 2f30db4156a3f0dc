// out[M,N] = epilogue((A[M,K] . W[N,K]^T) * sa[m] * sw[n] + bias[n]): rows and weights held as 8-bit codes with a scale a row of each.
// The products and their sums are whole numbers in 32 bits, so they are exact in any order; they are turned to 32-bit numbers once, at the end.
// (K is at most 133136: (2^31 - 1) / 127^2 is 133144, beyond which a sum could leave 32 bits.)
#include "common.cuh"

using namespace kvad;

KVAD_DEFINE_LAST_ERROR()

namespace {

template <typename T, int EPI>
__device__ __forceinline__ void put(void* out, int64_t at, float t) {
  if (EPI == EPI_GELU_TANH) t = gelu_tanh(t);
  if (EPI == EPI_GELU_ERF) t = gelu_erf(t);
  if (EPI == EPI_RESIDUAL) reinterpret_cast<float*>(out)[at] += t;
  else if (EPI == EPI_STORE_F32) reinterpret_cast<float*>(out)[at] = t;
  else reinterpret_cast<T*>(out)[at] = from_f32<T>(t);
}

// 64 x 64 outputs a block, 4 x 4 a thread; 64 entries of K at a time.
template <typename T, int EPI>
__global__ void __launch_bounds__(256)
linear_int8_kernel(const int8_t* __restrict__ a, int64_t lda, const float* __restrict__ sa, const int8_t* __restrict__ w, const float* __restrict__ sw,
                   const void* __restrict__ bias, int bias_f32, void* __restrict__ out, int64_t ldo, int M, int N, int K) {
  __shared__ int as[64][17], ws[64][17];
  pdl_launch_dependents();
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  int acc[4][4] = {};
  pdl_wait();
  for (int k0 = 0; k0 < K; k0 += 64) {
    const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
    int4 va = make_int4(0, 0, 0, 0), vw = va;
    if (m0 + r < M && k0 + c < K) va = *reinterpret_cast<const int4*>(a + (int64_t)(m0 + r) * lda + k0 + c);
    if (n0 + r < N && k0 + c < K) vw = *reinterpret_cast<const int4*>(w + (int64_t)(n0 + r) * K + k0 + c);
    __syncthreads();
    as[r][c / 4] = va.x; as[r][c / 4 + 1] = va.y; as[r][c / 4 + 2] = va.z; as[r][c / 4 + 3] = va.w;
    ws[r][c / 4] = vw.x; ws[r][c / 4 + 1] = vw.y; ws[r][c / 4 + 2] = vw.z; ws[r][c / 4 + 3] = vw.w;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(as[ty + 16 * i][k], ws[tx + 16 * j][k], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + ty + 16 * i;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx + 16 * j;
      if (m < M && n < N) {
        float t = (float)acc[i][j] * sa[m] * sw[n];
        if (bias != nullptr) t += load_param(bias, n, bias_f32);
        put<T, EPI>(out, (int64_t)m * ldo + n, t);
      }
    }
  }
}

template <typename T>
cudaError_t by_epilogue(int epi, dim3 grid, cudaStream_t stream, const int8_t* a, int64_t lda, const float* sa, const int8_t* w, const float* sw, const void* bias,
                        int bias_f32, void* out, int64_t ldo, int M, int N, int K) {
  auto go = [&](auto kernel) { return kvad_launch(kernel, grid, dim3(256), 0, stream, a, lda, sa, w, sw, bias, bias_f32, out, ldo, M, N, K); };
  switch (epi) {
    case EPI_STORE: return go(linear_int8_kernel<T, EPI_STORE>);
    case EPI_GELU_TANH: return go(linear_int8_kernel<T, EPI_GELU_TANH>);
    case EPI_GELU_ERF: return go(linear_int8_kernel<T, EPI_GELU_ERF>);
    case EPI_RESIDUAL: return go(linear_int8_kernel<T, EPI_RESIDUAL>);
    default: return go(linear_int8_kernel<T, EPI_STORE_F32>);
  }
}

}  // namespace

KVAD_EXPORT int kvad_linear_int8(int dtype, const int8_t* a, int64_t lda, const float* sa, const int8_t* w, const float* sw, const void* bias, int bias_f32,
                                 void* out, int64_t ldo, int M, int N, int K, int epi, cudaStream_t stream) {
  KVAD_REQUIRE(M > 0 && N > 0 && K > 0, "linear_int8: needs rows, outputs and inputs, got %d, %d, %d", M, N, K);
  if (K % 16 || K > 133136) KVAD_FAIL(KVAD_ERR_UNSUPPORTED, "linear_int8: inputs of a multiple of 16 entries up to 133136, not %d", K);
  KVAD_REQUIRE(((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(w)) & 15) == 0 && lda % 16 == 0,
               "linear_int8: rows and weights must start on 16-byte boundaries");
  KVAD_REQUIRE(epi >= EPI_STORE && epi <= EPI_STORE_F32, "linear_int8: unknown epilogue %d", epi);
  const dim3 grid((N + 63) / 64, (M + 63) / 64);
  KVAD_REQUIRE(grid.y <= 65535, "linear_int8: more rows than a launch takes");
  const cudaError_t e = dtype == KVAD_DTYPE_F32 ? by_epilogue<float>(epi, grid, stream, a, lda, sa, w, sw, bias, bias_f32, out, ldo, M, N, K)
                                                : by_epilogue<__nv_bfloat16>(epi, grid, stream, a, lda, sa, w, sw, bias, bias_f32, out, ldo, M, N, K);
  if (e != cudaSuccess) KVAD_FAIL(KVAD_ERR_CUDA, "linear_int8: launch failed: %s", cudaGetErrorString(e));
  KVAD_CHECK_LAUNCH("linear_int8");
  return KVAD_OK;
}
