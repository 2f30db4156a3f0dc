// Causal attention over the paged cache of 8-bit codes: key j of a head is kc_j ks_j and its value vc_j vs_j (codes times a scale each), and a row
// at position i of its sequence gets
//
//   out_i = sum_j w_ij vs_j vc_j / sum_j w_ij,    w_ij = exp(scale ks_j (q_i . kc_j) - max_j(...)),
//
// j over the positions that i sees: j <= i, and with a window i - j < window or j < keep_first.  The codes go into the products as they are (they are
// whole numbers) and the scales come in on the scores and the weights: one number a key, not one an entry.  Scores, maxima, sums and outputs are 32-bit.
//
// The general kernel: a warp has one row and head and walks 32 keys at a time, a lane a key for the scores, then a lane a few entries of the output.
#include "common.cuh"

using namespace kvad;

KVAD_DEFINE_LAST_ERROR()

namespace {

constexpr int PAGE = 64;
constexpr int MAX_HD = 256;

struct Cache {
  const int8_t* k;      // [pages, kv heads, 64, hd]
  const float* ks;      // [pages, kv heads, 64]
  const int8_t* v;
  const float* vs;
  const int* table;     // [sequences, width]
  int width, kv_heads, hd;
};

__device__ __forceinline__ float sum16(int4 c, const float* q) {
  const int w[4] = {c.x, c.y, c.z, c.w};
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s = fmaf((float)(int8_t)(w[i >> 2] >> (8 * (i & 3))), q[i], s);
  return s;
}

template <typename T>
__global__ void __launch_bounds__(128)
attention_int8_rows_kernel(const T* __restrict__ q, int64_t ld_q, T* __restrict__ out, int64_t ld_o, const int* __restrict__ seq_starts,
                           const int* __restrict__ kv_lens, Cache c, int n_rows, int n_seqs, int n_heads, float scale, int window, int keep_first) {
  __shared__ float q_sh[4][MAX_HD];
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + warp;
  pdl_wait();
  if (item >= (int64_t)n_rows * n_heads) return;
  const int row = (int)(item / n_heads), head = (int)(item - (int64_t)row * n_heads);
  const int kv = head / (n_heads / c.kv_heads), hd = c.hd;
  int lo = 0, hi = n_seqs;                    // the sequence whose rows hold this one: the last that starts at or before it
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (seq_starts[mid] <= row) lo = mid; else hi = mid;
  }
  const int seq = lo;
  const int pos = kv_lens[seq] - (seq_starts[seq + 1] - row);
  const int* table = c.table + (int64_t)seq * c.width;
  for (int j = lane; j < hd; j += 32) q_sh[warp][j] = to_f32(q[(int64_t)row * ld_q + head * hd + j]) * scale;
  __syncwarp();
  float o[MAX_HD / 32] = {};
  float top = -INFINITY, sum = 0.f;
  const int first = window > 0 && pos - window + 1 > 0 ? pos - window + 1 : 0;      // the window's first position
  const int kept = first < keep_first ? first : keep_first;
  for (int part = 0; part < 2; ++part) {
    const int begin = part ? first : 0, end = part ? pos + 1 : kept;
    for (int j0 = begin; j0 < end; j0 += 32) {
      const int j = j0 + lane;
      float s = -INFINITY, vs = 0.f;
      if (j < end) {
        const int64_t cell = ((int64_t)table[j / PAGE] * c.kv_heads + kv) * PAGE + j % PAGE;
        const int8_t* k = c.k + cell * hd;
        s = 0.f;
        for (int d = 0; d < hd; d += 16) s += sum16(*reinterpret_cast<const int4*>(k + d), q_sh[warp] + d);
        s *= c.ks[cell];
        vs = c.vs[cell];
      }
      const float new_top = fmaxf(top, warp_max(s));
      const float keep = new_top == -INFINITY ? 1.f : expf(top - new_top);
      const float p = s == -INFINITY ? 0.f : expf(s - new_top);
      sum = sum * keep + warp_sum(p);
      top = new_top;
      const float pv = p * vs;
      float t[MAX_HD / 32] = {};              // the tile's own sum, so that a chain of additions is as long as a tile and not as the context
      const int m = end - j0 < 32 ? end - j0 : 32;
      for (int x = 0; x < m; ++x) {
        const float px = __shfl_sync(0xffffffffu, pv, x);
        const int jj = j0 + x;
        const int8_t* v = c.v + (((int64_t)table[jj / PAGE] * c.kv_heads + kv) * PAGE + jj % PAGE) * hd;
#pragma unroll
        for (int i = 0; i < MAX_HD / 32; ++i)
          if (lane + 32 * i < hd) t[i] = fmaf(px, (float)v[lane + 32 * i], t[i]);
      }
#pragma unroll
      for (int i = 0; i < MAX_HD / 32; ++i) o[i] = fmaf(o[i], keep, t[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < MAX_HD / 32; ++i)
    if (lane + 32 * i < hd) out[(int64_t)row * ld_o + head * hd + lane + 32 * i] = from_f32<T>(o[i] / sum);
}

}  // namespace

KVAD_EXPORT int kvad_attention_int8(int dtype, const void* q, int64_t ld_q, void* out, int64_t ld_o, const int* seq_starts, const int* kv_lens,
                                    const int* table, int table_width, const int8_t* k_pages, const float* k_scales, const int8_t* v_pages,
                                    const float* v_scales, int n_rows, int n_seqs, int max_new, int n_heads, int kv_heads, int hd, int page, float scale,
                                    int window, int keep_first, cudaStream_t stream) {
  KVAD_REQUIRE(n_rows > 0 && n_seqs > 0 && max_new > 0 && table_width > 0, "attention_int8: needs rows, sequences and pages");
  KVAD_REQUIRE(n_heads > 0 && kv_heads > 0 && n_heads % kv_heads == 0, "attention_int8: %d heads do not divide into %d key/value heads", n_heads, kv_heads);
  if (hd <= 0 || hd % 16 || hd > MAX_HD) KVAD_FAIL(KVAD_ERR_UNSUPPORTED, "attention_int8: head sizes are multiples of 16 up to 256, not %d", hd);
  if (page != PAGE) KVAD_FAIL(KVAD_ERR_UNSUPPORTED, "attention_int8: pages hold 64 positions, not %d", page);
  KVAD_REQUIRE(((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15) == 0, "attention_int8: pages must start on a 16-byte boundary");
  KVAD_REQUIRE(window >= 0 && keep_first >= 0, "attention_int8: a window and kept first positions cannot be negative");
  const Cache c{k_pages, k_scales, v_pages, v_scales, table, table_width, kv_heads, hd};
  const int64_t blocks = ((int64_t)n_rows * n_heads + 3) / 4;
  KVAD_REQUIRE(blocks < (1ll << 31), "attention_int8: more rows and heads than a launch takes");
  auto go = [&](auto kernel, auto* qp, auto* op) {
    return kvad_launch(kernel, dim3((unsigned)blocks), dim3(128), 0, stream, qp, ld_q, op, ld_o, seq_starts, kv_lens, c, n_rows, n_seqs, n_heads, scale, window,
                       keep_first);
  };
  const cudaError_t e = dtype == KVAD_DTYPE_F32 ? go(attention_int8_rows_kernel<float>, (const float*)q, (float*)out)
                                                : go(attention_int8_rows_kernel<__nv_bfloat16>, (const __nv_bfloat16*)q, (__nv_bfloat16*)out);
  if (e != cudaSuccess) KVAD_FAIL(KVAD_ERR_CUDA, "attention_int8: launch failed: %s", cudaGetErrorString(e));
  KVAD_CHECK_LAUNCH("attention_int8");
  return KVAD_OK;
}
