// Keys and values held in the paged cache as 8-bit codes: every key and value of a position and head is a row of its own (codes of
// -127 .. 127 and a 32-bit scale, max |x| times the 32-bit 1/127; codes are x / scale rounded to the nearest integer, halves to the even one; a row of zeros has
// the scale 0, a row with a number that is not finite the scale NaN and codes 0).
//
//   pages   int8  [pages, kv heads, page size, head size]     a page of one head is one contiguous tile
//   scales  float [pages, kv heads, page size]                beside it
//
// so a position takes head size + 4 bytes a head, where bfloat16 takes 2 * head size.
//
// A group of lanes (a power of two, head size / 8 at least) has one row, and of it one head's keys or values, or several heads' where there are many rows: a lane
// brings eight entries, the group's maximum is a few shuffles, and the codes leave as eight bytes a lane.  Where a row goes is looked up once for these heads
// (a chain of two trips to memory), and all their entries are asked for before the first is worked on.  Bound by memory, entry + 1 bytes
// a code: 26289 bfloat16 rows of 8 heads of 128 are stored in 37 us (4.4 TB/s; four heads, turned to 32-bit on arrival: 41; four rows of one head a group: 79) and read in 30
// (5.5 TB/s).
//
// No pointer is __restrict__: what is promised not to change may be read before the wait for the kernel that writes it.
#include <type_traits>

#include "int8_codes.cuh"

using namespace kvad;

KVAD_DEFINE_LAST_ERROR()

namespace {

// Eight consecutive entries as they lie, and as floats; `vec`: on a boundary of 16 bytes.
template <typename T> struct Eight { uint4 w[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ void load8(const T* p, bool vec, Eight<T>& x) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) x.w[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    T* t = reinterpret_cast<T*>(&x);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = p[i];
  }
}
__device__ __forceinline__ void numbers(const Eight<float>& x, float* v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[4 * i] = __uint_as_float(x.w[i].x); v[4 * i + 1] = __uint_as_float(x.w[i].y); v[4 * i + 2] = __uint_as_float(x.w[i].z); v[4 * i + 3] = __uint_as_float(x.w[i].w);
  }
}
__device__ __forceinline__ void numbers(const Eight<__nv_bfloat16>& x, float* v) {
  const uint32_t w[4] = {x.w[0].x, x.w[0].y, x.w[0].z, x.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
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

struct Pages {
  const int* row_seq;
  const int* row_pos;
  const int* table;
  int width, heads, hd, page, shift;      // shift: log2 of the page size; negative: it is no power of two
  // Where the cache has row `row` and head `head`: (page * heads + head) * page size + place in the page.
  __device__ __forceinline__ int64_t cell(int row, int head) const {
    const int pos = row_pos[row], pg = shift >= 0 ? pos >> shift : pos / page;
    return ((int64_t)table[(int64_t)row_seq[row] * width + pg] * heads + head) * page + (pos - pg * page);
  }
};

// blockIdx.y: so many heads, blockIdx.z: their keys (0) or values (1).  Addresses step from head to head: worked out a head, they are half of the instructions.
template <typename T, int LANES, int R>
__global__ void __launch_bounds__(256, 4)
int8_store_kernel(const T* k_src, const T* v_src, int64_t ld_src, int vec, const Pages p, int8_t* k_pages,
                  float* k_scales, int8_t* v_pages, float* v_scales, int n) {
  pdl_launch_dependents();
  const int lane = threadIdx.x % LANES, row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, head = blockIdx.y * R;
  const int heads = row < n && lane * 8 < p.hd ? min(R, p.heads - head) : 0;
  const T* src = (blockIdx.z ? v_src : k_src) + row * ld_src + (head * p.hd + lane * 8);
  pdl_wait();
  Eight<T> x[R] = {};
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (i < heads) load8(src + i * p.hd, vec, x[i]);
  const int64_t cell = heads > 0 ? p.cell(row, head) : 0;
  int8_t* to = (blockIdx.z ? v_pages : k_pages) + cell * p.hd + lane * 8;
  float* scale = (blockIdx.z ? v_scales : k_scales) + cell;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float v[8], most = 0.f;
    numbers(x[i], v);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max_abs(most, v[e]);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) most = max_abs(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (i >= heads) continue;
    const Scale k = scale_of(__float_as_uint(most));
    *reinterpret_cast<uint2*>(to) = make_uint2(codes_of(v[0], v[1], v[2], v[3], k), codes_of(v[4], v[5], v[6], v[7], k));
    if (lane == 0) *scale = k.s;
    to += p.page * p.hd;
    scale += p.page;
  }
}

template <typename T, int LANES, int R>
__global__ void __launch_bounds__(256)
int8_load_kernel(T* k_out, T* v_out, int64_t ld_k, int64_t ld_v, int vec, const Pages p, const int8_t* k_pages,
                 const float* k_scales, const int8_t* v_pages, const float* v_scales, int n) {
  pdl_launch_dependents();
  const int lane = threadIdx.x % LANES, row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, head = blockIdx.y * R;
  pdl_wait();
  if (row >= n || lane * 8 >= p.hd) return;
  const int heads = min(R, p.heads - head);
  const int64_t cell = p.cell(row, head);
  const int8_t* from = (blockIdx.z ? v_pages : k_pages) + cell * p.hd + lane * 8;
  const float* scale = (blockIdx.z ? v_scales : k_scales) + cell;
  T* out = (blockIdx.z ? v_out : k_out) + row * (blockIdx.z ? ld_v : ld_k) + (head * p.hd + lane * 8);
  uint2 q[R];
  float s[R];
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (i < heads) {
      q[i] = *reinterpret_cast<const uint2*>(from + i * (p.page * p.hd));
      s[i] = scale[i * p.page];
    }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i >= heads) continue;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)((e < 4 ? q[i].x : q[i].y) >> (8 * (e & 3))) * s[i];
    store8(out + i * p.hd, vec, v);
  }
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
  KVAD_REQUIRE(heads <= 32767, "%s: more heads than a launch takes", what);
  if (hd <= 0 || hd % 16 || hd > 256) KVAD_FAIL(KVAD_ERR_UNSUPPORTED, "%s: head sizes are multiples of 16 up to 256, not %d", what, hd);
  KVAD_REQUIRE(((reinterpret_cast<uintptr_t>(kp) | reinterpret_cast<uintptr_t>(vp)) & 15) == 0, "%s: pages must start on a 16-byte boundary", what);
  return KVAD_OK;
}

constexpr int MANY = 512;        // rows from which on a group of lanes takes several heads of its row

Pages pages(const int* row_seq, const int* row_pos, const int* table, int width, int heads, int hd, int page) {
  int shift = -1;
  if ((page & (page - 1)) == 0)
    for (shift = 0; (1 << shift) < page;) ++shift;
  return Pages{row_seq, row_pos, table, width, heads, hd, page, shift};
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
  const Pages p = pages(row_seq, row_pos, table, table_width, heads, hd, page);
  const cudaError_t e = by_lanes(hd, [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    auto launch = [&](auto kernel, int r, auto* k, auto* v) {
      return kvad_launch(kernel, dim3((unsigned)((n + 256 / L - 1) / (256 / L)), (heads + r - 1) / r, 2), dim3(256), 0, stream, k, v, ld_src, vec, p, k_pages, k_scales,
                         v_pages, v_scales, n);
    };
    auto go = [&](auto* k, auto* v) {
      using T = std::remove_cv_t<std::remove_pointer_t<decltype(k)>>;
      constexpr int R = sizeof(T) == 2 ? 8 : 4;              // (128 bytes a lane)
      return n >= MANY ? launch(int8_store_kernel<T, L, R>, R, k, v) : launch(int8_store_kernel<T, L, 1>, 1, k, v);
    };
    return dtype == KVAD_DTYPE_F32 ? go((const float*)k_src, (const float*)v_src) : go((const __nv_bfloat16*)k_src, (const __nv_bfloat16*)v_src);
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
  const Pages p = pages(row_seq, row_pos, table, table_width, heads, hd, page);
  const cudaError_t e = by_lanes(hd, [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    auto launch = [&](auto kernel, int r, auto* k, auto* v) {
      return kvad_launch(kernel, dim3((unsigned)((n + 256 / L - 1) / (256 / L)), (heads + r - 1) / r, 2), dim3(256), 0, stream, k, v, ld_k, ld_v, vec, p, k_pages, k_scales,
                         v_pages, v_scales, n);
    };
    auto go = [&](auto* k, auto* v) {
      using T = std::remove_pointer_t<decltype(k)>;
      return n >= MANY ? launch(int8_load_kernel<T, L, 4>, 4, k, v) : launch(int8_load_kernel<T, L, 1>, 1, k, v);
    };
    return dtype == KVAD_DTYPE_F32 ? go((float*)k_out, (float*)v_out) : go((__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out);
  });
  if (e != cudaSuccess) KVAD_FAIL(KVAD_ERR_CUDA, "kv_read_int8: launch failed: %s", cudaGetErrorString(e));
  KVAD_CHECK_LAUNCH("kv_read_int8");
  return KVAD_OK;
}
