// out[M,N] = epilogue((A[M,K] . W[N,K]^T) * sa[m] * sw[n] + bias[n]): rows and weights held as 8-bit codes with a scale a row of each.
// The products and their sums are whole numbers in 32 bits, so they are exact in any order; they are turned to 32-bit numbers once, at the end.
// (K is at most 133136: (2^31 - 1) / 127^2 is 133144, beyond which a sum could leave 32 bits.)
//
// Many rows: the 5th-generation tensor cores (tcgen05.mma.kind::i8, 32-bit whole-number accumulators in tensor memory).  Both operands are K-major
// and come by TMA in blocks of 128 entries of K (one row of the 128-byte swizzle); a CTA computes tiles of 128 x BN, one after another, the
// epilogue of one under the products of the next (two accumulators).
//
// Few rows: a stream of weights.  A CTA has 16 outputs; its warps share K in pieces of 64 entries, of which a lane brings 16 contiguous
// bytes of two outputs' weights straight into registers - mma.sync takes K in any order, so long as rows and weights agree on it.
//
// Every wait on an mbarrier is bounded; one that runs out raises a counter (kvad_linear_int8_status), and the CTA frees its tensor memory and returns.
#include <type_traits>

#include "common.cuh"
#include "tcgen05.cuh"

using namespace kvad;

KVAD_DEFINE_LAST_ERROR()

namespace {

bool g_skip_copy = false;           // tests: the next launch of the tensor-core kernel leaves out its blocks' first copy

struct Out {
  void* p;
  int64_t ld;
  const float* sa;
  const float* sw;
  const void* bias;
  int bias_f32;
};

// tanh-form GELU as t / (1 + exp(-2u)): with u = c (t + 0.044715 t^3), (1 + tanh u) / 2 = 1 / (1 + exp(-2u)).  Good to a few units in the last place of 32 bits:
// the exponential's and the division's errors are relative, and nothing cancels.
__device__ __forceinline__ float gelu_tanh_logistic(float t) {
  const float c = 0.79788456f;
  const float e = __expf(-2.f * c * (t + 0.044715f * t * t * t));
  return __fdividef(t, 1.f + e);
}

template <int EPI> __device__ __forceinline__ float finish(float t) {
  if (EPI == EPI_GELU_TANH) {
    const float g = gelu_tanh_logistic(t);
    return t < -10.f ? 0.f * t : g;         // (there the result is below 2^-120, exp(-2u) passes 2^126, and t^3 may leave 32 bits)
  }
  if (EPI == EPI_GELU_ERF) return gelu_erf(t);
  return t;
}

template <typename T, int EPI>
__device__ __forceinline__ void put(const Out& o, int64_t at, float t) {
  if (EPI == EPI_RESIDUAL) reinterpret_cast<float*>(o.p)[at] += t;
  else if (EPI == EPI_STORE_F32) reinterpret_cast<float*>(o.p)[at] = t;
  else reinterpret_cast<T*>(o.p)[at] = from_f32<T>(t);
}

// ---------------------------------------------------------------------------------------------------------------------------
// Few rows
// ---------------------------------------------------------------------------------------------------------------------------
constexpr int FEW_WARPS = 8;

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT groups of eight rows.  Weights are the M side of the product (16 outputs), rows its N side.
// (`a` is not __restrict__: what is promised not to change may be read before the wait for the kernel that writes it.)
template <typename T, int EPI, int NT>
__global__ void __launch_bounds__(FEW_WARPS * 32)
linear_int8_few_kernel(const int8_t* a, int64_t lda, const int8_t* __restrict__ w, Out o, int M, int N, int K) {
  __shared__ int part[FEW_WARPS][NT * 8][17];
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16;
  const int chunks = (K + 63) / 64;
  constexpr int U = NT <= 2 ? 4 : 2;            // pieces of K a lane asks for at a time
  int acc[NT][4] = {};
  const int8_t* w0 = w + (int64_t)(n0 + g < N ? n0 + g : N - 1) * K + t * 16;
  const int8_t* w1 = w + (int64_t)(n0 + g + 8 < N ? n0 + g + 8 : N - 1) * K + t * 16;
  bool waited = false;
  for (int c0 = warp; c0 < chunks; c0 += FEW_WARPS * U) {
    int4 wa[U], wb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (c0 + u * FEW_WARPS) * 64;
      wa[u] = wb[u] = make_int4(0, 0, 0, 0);
      if (k + t * 16 < K) {
        wa[u] = __ldg(reinterpret_cast<const int4*>(w0 + k));
        wb[u] = __ldg(reinterpret_cast<const int4*>(w1 + k));
      }
    }
    if (!waited) {                              // weights do not depend on the kernel before
      pdl_wait();
      waited = true;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (c0 + u * FEW_WARPS) * 64 + t * 16;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int m = nt * 8 + g;
        int4 x = make_int4(0, 0, 0, 0);
        if (m < M && k < K) x = *reinterpret_cast<const int4*>(a + (int64_t)m * lda + k);
        mma_s8(acc[nt], wa[u].x, wb[u].x, wa[u].y, wb[u].y, x.x, x.y);
        mma_s8(acc[nt], wa[u].z, wb[u].z, wa[u].w, wb[u].w, x.z, x.w);
      }
    }
  }
  if (!waited) pdl_wait();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {             // accumulator: outputs g and g + 8, rows 2t and 2t + 1
    part[warp][nt * 8 + 2 * t][g] = acc[nt][0];
    part[warp][nt * 8 + 2 * t + 1][g] = acc[nt][1];
    part[warp][nt * 8 + 2 * t][g + 8] = acc[nt][2];
    part[warp][nt * 8 + 2 * t + 1][g + 8] = acc[nt][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 8 * 16; i += FEW_WARPS * 32) {
    const int m = i >> 4, j = i & 15, n = n0 + j;
    if (m >= M || n >= N) continue;
    int s = 0;
#pragma unroll
    for (int x = 0; x < FEW_WARPS; ++x) s += part[x][m][j];
    float y = (float)s * o.sa[m] * o.sw[n];
    if (o.bias != nullptr) y += load_param(o.bias, n, o.bias_f32);
    put<T, EPI>(o, (int64_t)m * o.ld + n, finish<EPI>(y));
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Many rows
// ---------------------------------------------------------------------------------------------------------------------------
constexpr int BM = 128, BK = 128;             // 128 entries of K: one row of the 128-byte swizzle
constexpr int THREADS = 320;                  // warp 0: TMA, warp 1: products and tensor memory, warps 2-9: epilogue

template <int BN> struct Tile {
  static constexpr uint32_t A_BYTES = BM * BK, B_BYTES = BN * BK;
  static constexpr int STAGES_RAW = 192 * 1024 / (A_BYTES + B_BYTES);
  static constexpr int STAGES = STAGES_RAW > 8 ? 8 : STAGES_RAW;
  static constexpr uint32_t OFF_SLAB = STAGES * (A_BYTES + B_BYTES);        // 4 KB an epilogue warp: 32 rows x 128 bytes of output on their way out by TMA
  static constexpr uint32_t OFF_BAR = OFF_SLAB + 8 * 4096;
  static constexpr size_t SMEM = OFF_BAR + (2 * STAGES + 4) * 8 + 16 + 1024;
};

// Whole-number products of 8-bit codes with a 32-bit accumulator: both operands signed, both K-major.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  const uint32_t zero = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
      ::"r"(d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(zero) : "memory");
}

// Sixteen columns of a row from tensor memory, there when the statement is over.  (One statement for the load and the wait: between two, the compiler is free to work on
// registers that are still on their way.)
__device__ __forceinline__ void tmem_read16(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(addr) : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// Sixteen consecutive entries of a vector from `n` on, zeros beyond N.
__device__ __forceinline__ void load16(const float* p, int n, int N, float* v) {
  if (n + 16 <= N && (reinterpret_cast<uintptr_t>(p + n) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(p + n) + i);
      v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = n + i < N ? __ldg(p + n + i) : 0.f;
  }
}

// One row's sixteen consecutive outputs where TMA cannot take them (a base or row stride off 16 bytes).
template <typename T, int EPI>
__device__ __forceinline__ void put16(const Out& o, int row, int n, int N, const float* v) {
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (n + j < N) put<T, EPI>(o, (int64_t)row * o.ld + n + j, v[j]);
}

template <typename T, int EPI, int BN>
__global__ void __launch_bounds__(THREADS, 1)
linear_int8_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_out,
                   int tma_out, Out o, int M, int N, int K, int skip_copy) {
  using L = Tile<BN>;
  constexpr int STAGES = L::STAGES;
  constexpr uint32_t TMEM = 2 * BN;             // two accumulators (a power of two)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* a_tiles = smem;
  uint8_t* b_tiles = smem + STAGES * L::A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;          // [2] the accumulator is complete
  uint64_t* acc_empty = acc_full + 2;           // [2] the eight epilogue warps have read it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  __shared__ int gave_up;

  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_n = (N + BN - 1) / BN, n_tiles = tiles_n * ((M + BM - 1) / BM), n_kb = (K + BK - 1) / BK;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_a);
    prefetch_tensormap(&map_w);
    if (tma_out) prefetch_tensormap(&map_out);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 8);
    }
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(tmem_slot, TMEM);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;                          // stages filled so far, over all tiles
      int asked = 0;                            // of the first tile: weights on the way before the kernel before has finished
      for (int t = blockIdx.x; t < n_tiles && ok; t += gridDim.x) {
        const int n0 = t % tiles_n * BN, m0 = t / tiles_n * BM;
        if (t == (int)blockIdx.x) {
          asked = n_kb < STAGES ? n_kb : STAGES;
          for (int i = 0; i < asked; ++i) {
            mbar_expect_tx(&full[i], L::A_BYTES + L::B_BYTES);
            if (!(skip_copy && i == 0)) tma_load_2d(b_tiles + i * L::B_BYTES, &map_w, &full[i], i * BK, n0);
          }
          pdl_wait();
          for (int i = 0; i < asked; ++i) tma_load_2d(a_tiles + i * L::A_BYTES, &map_a, &full[i], i * BK, m0);
          it = asked;
        }
        for (int i = t == (int)blockIdx.x ? asked : 0; i < n_kb; ++i, ++it) {
          const int s = it % STAGES;
          if (it >= (uint32_t)STAGES && !mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1)) { ok = false; break; }
          mbar_expect_tx(&full[s], L::A_BYTES + L::B_BYTES);
          tma_load_2d(a_tiles + s * L::A_BYTES, &map_a, &full[s], i * BK, m0);
          tma_load_2d(b_tiles + s * L::B_BYTES, &map_w, &full[s], i * BK, n0);
        }
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_i8(BM, BN);
    const bool one = elect_one();
    const uint64_t a_desc0 = sw128_desc(smem_u32(a_tiles)), b_desc0 = sw128_desc(smem_u32(b_tiles));
    uint32_t it = 0;
    int lt = 0;                                 // tiles of this CTA so far
    for (int t = blockIdx.x; t < n_tiles && ok; t += gridDim.x, ++lt) {
      const int buf = lt & 1;
      if (lt >= 2) {
        ok = mbar_wait(&acc_empty[buf], ((lt >> 1) & 1) ^ 1);
        if (!ok) break;
        tc_fence_after();
      }
      const uint32_t acc = tmem + (uint32_t)(buf * BN);
      for (int i = 0; i < n_kb; ++i, ++it) {
        const int s = it % STAGES;
        ok = mbar_wait(&full[s], (it / STAGES) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint64_t a_desc = a_desc0 + (uint32_t)s * (L::A_BYTES >> 4), b_desc = b_desc0 + (uint32_t)s * (L::B_BYTES >> 4);
        if (one) {
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)     // 32 entries further along K: 32 bytes inside the swizzled row
            umma_i8(acc, a_desc + (uint64_t)(k * 2), b_desc + (uint64_t)(k * 2), idesc, (i > 0 || k > 0) ? 1u : 0u);
          umma_commit(&empty[s]);
        }
      }
      if (ok && one) umma_commit(&acc_full[buf]);
    }
  } else {
    const int quarter = warp & 3, half = warp >= 6 ? 1 : 0;       // two warps share a quarter of the lanes and take its slabs in turn
    constexpr bool F32_OUT = EPI == EPI_RESIDUAL || EPI == EPI_STORE_F32 || std::is_same<T, float>::value;
    constexpr int SLAB = F32_OUT ? 32 : 64;     // 128 bytes of output a row
    uint8_t* slab = smem + L::OFF_SLAB + (warp - 2) * 4096;
    bool used = false;
    int lt = 0;
    pdl_wait();
    for (int t = blockIdx.x; t < n_tiles && ok; t += gridDim.x, ++lt) {
      const int n0 = t % tiles_n * BN, m0 = t / tiles_n * BM, buf = lt & 1;
      const int row = m0 + quarter * 32 + lane;
      const float sa = row < M ? o.sa[row] : 0.f;
      if (!mbar_wait(&acc_full[buf], (lt >> 1) & 1)) { ok = false; break; }
      tc_fence_after();
      const uint32_t acc = tmem + (uint32_t)(buf * BN) + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
      for (int c0 = half * SLAB; c0 < BN; c0 += 2 * SLAB) {
        if (n0 + c0 >= N) break;
        if (tma_out && used) {                  // the slab's last journey has been read
          if (lane == 0) bulk_wait_read();
          __syncwarp();
        }
        used = true;
#pragma unroll
        for (int cc = 0; cc < SLAB; cc += 16) {
          float v[16], s[16];
          load16(o.sw, n0 + c0 + cc, N, s);
          tmem_read16(acc + (uint32_t)(c0 + cc), v);
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = (float)__float_as_int(v[j]) * sa * s[j];
          if (o.bias != nullptr) {
            if (o.bias_f32) {
              load16(reinterpret_cast<const float*>(o.bias), n0 + c0 + cc, N, s);
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j) s[j] = n0 + c0 + cc + j < N ? load_param(o.bias, n0 + c0 + cc + j, 0) : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] += s[j];
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = finish<EPI>(v[j]);
          if (!tma_out) {
            if (row < M) put16<T, EPI>(o, row, n0 + c0 + cc, N, v);
          } else if (F32_OUT) {
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<float4*>(slab + lane * 128 + ((((cc + j) >> 2) ^ (lane & 7)) << 4)) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 16; j += 8) {
              uint32_t q[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                __nv_bfloat162 p = __floats2bfloat162_rn(v[j + 2 * e], v[j + 2 * e + 1]);
                q[e] = *reinterpret_cast<uint32_t*>(&p);
              }
              *reinterpret_cast<uint4*>(slab + lane * 128 + ((((cc + j) >> 3) ^ (lane & 7)) << 4)) = make_uint4(q[0], q[1], q[2], q[3]);
            }
          }
        }
        if (tma_out) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && m0 + quarter * 32 < M) {
            if (EPI == EPI_RESIDUAL) tma_reduce_add_2d(&map_out, slab, n0 + c0, m0 + quarter * 32);
            else tma_store_2d(&map_out, slab, n0 + c0, m0 + quarter * 32);
            bulk_commit();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_one(&acc_empty[buf]);
    }
    if (lane == 0) bulk_wait_all();
  }
  if (!ok) gave_up = 1;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (gave_up) outlast_what_is_in_flight();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, TMEM);
  }
}

int sm_count() {
  static int n = 0;
  if (n == 0) {
    int dev = 0, v = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && v > 0) n = v;
    else n = 148;
  }
  return n;
}

// A matrix whose rows lie ld entries apart, `box_rows` x 128 bytes a copy.
int tensor_map(const void* p, CUtensorMapDataType type, int size, int64_t ld, int rows, int cols, int box_rows, CUtensorMap* map) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) KVAD_FAIL(KVAD_ERR_CUDA, "linear_int8: the driver does not offer cuTensorMapEncodeTiled");
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * size};
  cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows}, elem[2] = {1, 1};
  CUresult r = fn(map, type, 2, const_cast<void*>(p), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) KVAD_FAIL(KVAD_ERR_CUDA, "linear_int8: cuTensorMapEncodeTiled failed (%d) for [%d, %d] entries, %lld apart", (int)r, rows, cols, (long long)ld);
  return KVAD_OK;
}

template <typename T, int EPI, int BN>
int many(const int8_t* a, int64_t lda, const int8_t* w, const Out& o, int M, int N, int K, cudaStream_t stream) {
  using L = Tile<BN>;
  CUtensorMap ma, mw, mo;
  int rc = tensor_map(a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, lda, M, K, BM, &ma);
  if (rc == KVAD_OK) rc = tensor_map(w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, N, K, BN, &mw);
  if (rc != KVAD_OK) return rc;
  constexpr bool f32_out = EPI == EPI_RESIDUAL || EPI == EPI_STORE_F32 || std::is_same<T, float>::value;
  constexpr int size = f32_out ? 4 : 2;
  const int tma_out = (o.ld * size) % 16 == 0 && (reinterpret_cast<uintptr_t>(o.p) & 15) == 0;
  if (tma_out) rc = tensor_map(o.p, f32_out ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, size, o.ld, M, N, 32, &mo);
  else mo = ma;
  if (rc != KVAD_OK) return rc;
  auto kernel = linear_int8_kernel<T, EPI, BN>;
  static bool configured = false;
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::SMEM);
    if (e != cudaSuccess) KVAD_FAIL(KVAD_ERR_CUDA, "linear_int8: cannot reserve %zu bytes of shared memory: %s", L::SMEM, cudaGetErrorString(e));
    configured = true;
  }
  const int64_t n_tiles = (int64_t)((N + BN - 1) / BN) * ((M + BM - 1) / BM);
  KVAD_REQUIRE(n_tiles < (1ll << 30), "linear_int8: %lld tiles are more than one launch takes", (long long)n_tiles);
  const int skip = g_skip_copy;
  g_skip_copy = false;
  const cudaError_t e = kvad_launch(kernel, dim3((unsigned)(n_tiles < sm_count() ? n_tiles : sm_count())), dim3(THREADS), L::SMEM, stream, ma, mw, mo, tma_out, o, M,
                                    N, K, skip);
  if (e != cudaSuccess) KVAD_FAIL(KVAD_ERR_CUDA, "linear_int8: launch failed: %s", cudaGetErrorString(e));
  return KVAD_OK;
}

template <typename T, int EPI>
int few(const int8_t* a, int64_t lda, const int8_t* w, const Out& o, int M, int N, int K, cudaStream_t stream) {
  auto go = [&](auto kernel) { return kvad_launch(kernel, dim3((N + 15) / 16), dim3(FEW_WARPS * 32), 0, stream, a, lda, w, o, M, N, K); };
  const cudaError_t e = M <= 8 ? go(linear_int8_few_kernel<T, EPI, 1>) : M <= 16 ? go(linear_int8_few_kernel<T, EPI, 2>)
                        : M <= 32 ? go(linear_int8_few_kernel<T, EPI, 4>) : go(linear_int8_few_kernel<T, EPI, 8>);
  if (e != cudaSuccess) KVAD_FAIL(KVAD_ERR_CUDA, "linear_int8: launch failed: %s", cudaGetErrorString(e));
  return KVAD_OK;
}

// The tile width whose waves of tiles over the SMs take the least: a wave of width BN takes BN's time, and a tile's start as much as 32 columns more; below 128
// columns the products wait for their rows from shared memory.
int tile_width(int M, int N) {
  int best = 0;
  int64_t best_cost = 0;
  for (int bn : {256, 128, 64}) {
    const int64_t tiles = (int64_t)((N + bn - 1) / bn) * ((M + BM - 1) / BM);
    const int64_t cost = (tiles + sm_count() - 1) / sm_count() * ((bn < 96 ? 96 : bn) + 32);
    if (best == 0 || cost < best_cost) best = bn, best_cost = cost;
  }
  return best;
}

constexpr int FEW_MAX = 64;

template <typename T, int EPI>
int go(const int8_t* a, int64_t lda, const int8_t* w, const Out& o, int M, int N, int K, int form, cudaStream_t stream) {
  if (form == 1 || (form == 0 && M <= FEW_MAX)) return few<T, EPI>(a, lda, w, o, M, N, K, stream);
  const int bn = form >= 64 ? form : tile_width(M, N);
  return bn == 256 ? many<T, EPI, 256>(a, lda, w, o, M, N, K, stream) : bn == 128 ? many<T, EPI, 128>(a, lda, w, o, M, N, K, stream)
                                                                                  : many<T, EPI, 64>(a, lda, w, o, M, N, K, stream);
}

}  // namespace

// `form`: 0: by the sizes; 1: the kernel of few rows (at most 64); 64, 128, 256: the kernel of many rows with tiles so wide.
KVAD_EXPORT int kvad_linear_int8(int dtype, const int8_t* a, int64_t lda, const float* sa, const int8_t* w, const float* sw, const void* bias, int bias_f32,
                                 void* out, int64_t ldo, int M, int N, int K, int epi, int form, cudaStream_t stream) {
  KVAD_REQUIRE(M > 0 && N > 0 && K > 0, "linear_int8: needs rows, outputs and inputs, got %d, %d, %d", M, N, K);
  if (K % 16 || K > 133136) KVAD_FAIL(KVAD_ERR_UNSUPPORTED, "linear_int8: inputs of a multiple of 16 entries up to 133136, not %d", K);
  KVAD_REQUIRE(((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(w)) & 15) == 0 && lda % 16 == 0,
               "linear_int8: rows and weights must start on 16-byte boundaries");
  KVAD_REQUIRE(epi >= EPI_STORE && epi <= EPI_STORE_F32, "linear_int8: unknown epilogue %d", epi);
  KVAD_REQUIRE(form == 0 || form == 64 || form == 128 || form == 256 || (form == 1 && M <= FEW_MAX), "linear_int8: no form %d for %d rows", form, M);
  const Out o{out, ldo, sa, sw, bias, bias_f32};
  int rc = KVAD_OK;
  const bool f32 = dtype == KVAD_DTYPE_F32;
  switch (epi) {
    case EPI_STORE: rc = f32 ? go<float, EPI_STORE_F32>(a, lda, w, o, M, N, K, form, stream) : go<__nv_bfloat16, EPI_STORE>(a, lda, w, o, M, N, K, form, stream); break;
    case EPI_GELU_TANH: rc = f32 ? go<float, EPI_GELU_TANH>(a, lda, w, o, M, N, K, form, stream) : go<__nv_bfloat16, EPI_GELU_TANH>(a, lda, w, o, M, N, K, form, stream); break;
    case EPI_GELU_ERF: rc = f32 ? go<float, EPI_GELU_ERF>(a, lda, w, o, M, N, K, form, stream) : go<__nv_bfloat16, EPI_GELU_ERF>(a, lda, w, o, M, N, K, form, stream); break;
    case EPI_RESIDUAL: rc = go<float, EPI_RESIDUAL>(a, lda, w, o, M, N, K, form, stream); break;
    default: rc = go<float, EPI_STORE_F32>(a, lda, w, o, M, N, K, form, stream);
  }
  if (rc != KVAD_OK) return rc;
  KVAD_CHECK_LAUNCH("linear_int8");
  return KVAD_OK;
}

// How many bounded waits have run out in this process (0 unless something is wrong).  Synchronises the device.
KVAD_EXPORT int kvad_linear_int8_status() {
  int n = 0;
  if (cudaMemcpyFromSymbol(&n, g_wait_timeouts, sizeof(n)) != cudaSuccess) return -1;
  return n;
}

// Tests of the bounded waits: `wait_limit` > 0 sets how many polls a wait makes before it gives up (0: the library's own limit); `skip_copy` leaves the first
// copy out of the NEXT launch's blocks (the kernel of many rows), so that the wait for it runs out.  Synchronises the device.
KVAD_EXPORT int kvad_linear_int8_test_hooks(unsigned wait_limit, int skip_copy) {
  g_skip_copy = skip_copy;
  return set_wait_limit(wait_limit);
}
