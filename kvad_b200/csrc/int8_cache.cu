// Keys and values held in the paged cache as 8-bit codes: every key and value of a position and head is a row of its own (codes of
// -127 .. 127 and a 32-bit scale, max |x| times the 32-bit 1/127; codes are x / scale rounded to the nearest integer, halves to the even one; a row of zeros has
// the scale 0, a row with a number that is not finite the scale NaN and codes 0).
//
//   pages   int8  [pages, kv heads, page size, head size]     a page of one head is one contiguous tile
//   scales  float [pages, kv heads, page size]                beside it
//
// so a position takes head size + 4 bytes a head, where bfloat16 takes 2 * head size.
//
// A group of lanes (a power of two, head size / 8 at least) has one row: a lane brings eight entries, the group's maximum is a few shuffles, and
// the codes leave as eight bytes a lane.  Keys and values go in one launch.  Bound by memory: 2 * (entry + 1) bytes a code, counting both directions.
#include <type_traits>

#include "common.cuh"

using namespace kvad;

KVAD_DEFINE_LAST_ERROR()

namespace {

// Eight consecutive entries as floats; `vec`: on a boundary of 16 bytes.
__device__ __forceinline__ void load8(const float* p, bool vec, float* v) {
  if (vec) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[i];
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, bool vec, float* v) {
  if (vec) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __bfloat162float(p[i]);
  }
}
__device__ __forceinline__ void store8(float* p, bool vec, const float* v) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = v[i];
  }
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, bool vec, const float* v) {
  if (vec) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __float2bfloat16_rn(v[i]);
  }
}

// Which row of the cache a group of lanes has: (token row, head, keys or values).  -1: none.
struct Place {
  int64_t row;       // of the token, in the packed rows
  int64_t cell;      // of the cache: (page * heads + head) * page size + place in the page
  int head;
  bool value;
};
__device__ __forceinline__ Place place_of(int64_t item, int heads, int page, const int* row_seq, const int* row_pos, const int* table, int table_width) {
  Place p;
  const int64_t rh = item >> 1;
  p.value = item & 1;
  p.row = rh / heads;
  p.head = (int)(rh - p.row * heads);
  const int pos = row_pos[p.row], pg = pos / page;
  const int id = table[(int64_t)row_seq[p.row] * table_width + pg];
  p.cell = ((int64_t)id * heads + p.head) * page + (pos - pg * page);
  return p;
}

template <typename T, int LANES>
__global__ void __launch_bounds__(256)
int8_store_kernel(const T* __restrict__ k_src, const T* __restrict__ v_src, int64_t ld_src, int vec, const int* __restrict__ row_seq,
                  const int* __restrict__ row_pos, const int* __restrict__ table, int table_width, int8_t* __restrict__ k_pages,
                  float* __restrict__ k_scales, int8_t* __restrict__ v_pages, float* __restrict__ v_scales, int n, int heads, int hd, int page) {
  pdl_launch_dependents();
  const int lane = threadIdx.x % LANES;
  const int64_t item = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  pdl_wait();
  const bool has = item < (int64_t)n * heads * 2;
  const bool in = has && lane * 8 < hd;
  Place p{};
  float v[8] = {};
  if (has) p = place_of(item, heads, page, row_seq, row_pos, table, table_width);
  if (in) load8((p.value ? v_src : k_src) + p.row * ld_src + (int64_t)p.head * hd + lane * 8, vec, v);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (!in) return;
  const bool finite = top < 0x7f800000u;
  const float scale = finite ? __fmul_rn(__uint_as_float(top), 1.f / 127.f) : __uint_as_float(0x7fffffffu);
  const bool some = finite && scale > 0.f;
  uint32_t w[2] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = some ? __fdiv_rn(v[i], scale) : 0.f;
    w[i >> 2] |= (uint32_t)(__float2int_rn(fminf(fmaxf(q, -127.f), 127.f)) & 0xff) << (8 * (i & 3));
  }
  *reinterpret_cast<uint2*>((p.value ? v_pages : k_pages) + p.cell * hd + lane * 8) = make_uint2(w[0], w[1]);
  if (lane == 0) (p.value ? v_scales : k_scales)[p.cell] = scale;
}

template <typename T, int LANES>
__global__ void __launch_bounds__(256)
int8_load_kernel(T* __restrict__ k_out, T* __restrict__ v_out, int64_t ld_k, int64_t ld_v, int vec, const int* __restrict__ row_seq,
                 const int* __restrict__ row_pos, const int* __restrict__ table, int table_width, const int8_t* __restrict__ k_pages,
                 const float* __restrict__ k_scales, const int8_t* __restrict__ v_pages, const float* __restrict__ v_scales, int n, int heads, int hd, int page) {
  pdl_launch_dependents();
  const int lane = threadIdx.x % LANES;
  const int64_t item = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  pdl_wait();
  if (item >= (int64_t)n * heads * 2 || lane * 8 >= hd) return;
  const Place p = place_of(item, heads, page, row_seq, row_pos, table, table_width);
  const uint2 q = *reinterpret_cast<const uint2*>((p.value ? v_pages : k_pages) + p.cell * hd + lane * 8);
  const float s = (p.value ? v_scales : k_scales)[p.cell];
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)(int8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3))) * s;
  store8((p.value ? v_out : k_out) + p.row * (p.value ? ld_v : ld_k) + (int64_t)p.head * hd + lane * 8, vec, v);
}

// f(lanes) with as many lanes as a row of hd entries takes, a power of two.
template <typename F> cudaError_t by_lanes(int hd, F f) {
  if (hd <= 16) return f(std::integral_constant<int, 2>());
  if (hd <= 32) return f(std::integral_constant<int, 4>());
  if (hd <= 64) return f(std::integral_constant<int, 8>());
  if (hd <= 128) return f(std::integral_constant<int, 16>());
  return f(std::integral_constant<int, 32>());
}

int check(const char* what, int n, int heads, int hd, int page, int table_width, const void* kp, const void* vp) {
  KVAD_REQUIRE(n > 0 && heads > 0 && page > 0 && table_width > 0, "%s: needs rows, heads and pages", what);
  if (hd <= 0 || hd % 16 || hd > 256) KVAD_FAIL(KVAD_ERR_UNSUPPORTED, "%s: head sizes are multiples of 16 up to 256, not %d", what, hd);
  KVAD_REQUIRE(((reinterpret_cast<uintptr_t>(kp) | reinterpret_cast<uintptr_t>(vp)) & 15) == 0, "%s: pages must start on a 16-byte boundary", what);
  return KVAD_OK;
}

bool whole(const void* p, int64_t ld, int size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld * size) % 16 == 0; }

}  // namespace

KVAD_EXPORT int kvad_kv_store_int8(int dtype, const void* k_src, const void* v_src, int64_t ld_src, const int* row_seq, const int* row_pos, const int* table,
                                   int table_width, int8_t* k_pages, float* k_scales, int8_t* v_pages, float* v_scales, int n, int heads, int hd, int page,
                                   cudaStream_t stream) {
  const int bad = check("kv_store_int8", n, heads, hd, page, table_width, k_pages, v_pages);
  if (bad) return bad;
  const int size = dtype == KVAD_DTYPE_F32 ? 4 : 2;
  const int vec = whole(k_src, ld_src, size) && whole(v_src, ld_src, size);
  const cudaError_t e = by_lanes(hd, [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    const int64_t blocks = ((int64_t)n * heads * 2 + 256 / L - 1) / (256 / L);
    if (blocks >= (1ll << 31)) return cudaErrorInvalidConfiguration;
    auto launch = [&](auto kernel, auto* k, auto* v) {
      return kvad_launch(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, k, v, ld_src, vec, row_seq, row_pos, table, table_width, k_pages, k_scales,
                         v_pages, v_scales, n, heads, hd, page);
    };
    return dtype == KVAD_DTYPE_F32 ? launch(int8_store_kernel<float, L>, (const float*)k_src, (const float*)v_src)
                                   : launch(int8_store_kernel<__nv_bfloat16, L>, (const __nv_bfloat16*)k_src, (const __nv_bfloat16*)v_src);
  });
  if (e != cudaSuccess) KVAD_FAIL(KVAD_ERR_CUDA, "kv_store_int8: launch failed: %s", cudaGetErrorString(e));
  KVAD_CHECK_LAUNCH("kv_store_int8");
  return KVAD_OK;
}

KVAD_EXPORT int kvad_kv_read_int8(int dtype, void* k_out, void* v_out, int64_t ld_k, int64_t ld_v, const int* row_seq, const int* row_pos, const int* table,
                                  int table_width, const int8_t* k_pages, const float* k_scales, const int8_t* v_pages, const float* v_scales, int n, int heads,
                                  int hd, int page, cudaStream_t stream) {
  const int bad = check("kv_read_int8", n, heads, hd, page, table_width, k_pages, v_pages);
  if (bad) return bad;
  const int size = dtype == KVAD_DTYPE_F32 ? 4 : 2;
  const int vec = whole(k_out, ld_k, size) && whole(v_out, ld_v, size);
  const cudaError_t e = by_lanes(hd, [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    const int64_t blocks = ((int64_t)n * heads * 2 + 256 / L - 1) / (256 / L);
    if (blocks >= (1ll << 31)) return cudaErrorInvalidConfiguration;
    auto launch = [&](auto kernel, auto* k, auto* v) {
      return kvad_launch(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, k, v, ld_k, ld_v, vec, row_seq, row_pos, table, table_width, k_pages, k_scales,
                         v_pages, v_scales, n, heads, hd, page);
    };
    return dtype == KVAD_DTYPE_F32 ? launch(int8_load_kernel<float, L>, (float*)k_out, (float*)v_out)
                                   : launch(int8_load_kernel<__nv_bfloat16, L>, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out);
  });
  if (e != cudaSuccess) KVAD_FAIL(KVAD_ERR_CUDA, "kv_read_int8: launch failed: %s", cudaGetErrorString(e));
  KVAD_CHECK_LAUNCH("kv_read_int8");
  return KVAD_OK;
}
