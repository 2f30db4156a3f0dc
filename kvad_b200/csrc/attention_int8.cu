// Causal attention over the paged cache of 8-bit codes: key j of a head is kc_j ks_j and its value vc_j vs_j (codes times a scale each), and a row
// at position i of its sequence gets
//
//   out_i = sum_j w_ij vs_j vc_j / sum_j w_ij,    w_ij = exp(scale ks_j (q_i . kc_j) - max_j(...)),
//
// j over the positions that i sees: j <= i, and with a window i - j < window or j < keep_first.
//
// A block has up to 16 rows - (token, head) pairs of one key/value head's group: the heads of a single token, or of a few - and a range of pages; its warps
// take the pages in turn, each with its own running maximum, sums and outputs, and they meet in shared memory at the end (and blocks of the same rows in
// `scratch`, which a second kernel reads).  Single tokens are bound by the bytes of the cache: every warp has a page of keys and one of values on their way
// (TMA, swizzled by their row's length) while it works on those before, so an SM has some 100 KB in flight.
//
// The products run on mma.sync in half precision with codes as they are (whole numbers, exact): a byte under 0x64 is 1024 + code + 128, less 1152.  A
// row's queries are brought to [1, 4) by a power of two, exactly, and in 32-bit go in two pieces (22 bits); the scales come in on the scores, which a thread has for two
// keys of eight.  Weights times their value's scale go in as half precision in one piece (11 bits; the output has 8), or two.  To keep them in range the exponent c of a
// page's largest value scale is kept apart: with t the score in powers of two,
//
//   p_ij = 2^(t_ij + c - r_i + 12),   out_i = sum_j (p_ij vs_j 2^-c) vc_j / sum_j p_ij 2^-c,   r_i the largest t + c seen so far.
//
// Scores, maxima, sums and outputs are 32-bit.
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "tcgen05.cuh"

using namespace kvad;

KVAD_DEFINE_LAST_ERROR()

namespace {

constexpr int PAGE = 64, ROWS = 16;
constexpr float LOG2E = 1.4426950408889634f, HEAD = 12.f;

bool g_skip_copy = false;                       // tests: the next launch's warps leave out their first page

struct Args {
  const void* q;
  int64_t ld_q;
  void* out;
  int64_t ld_out;
  const int* seq_starts;
  const int* kv_lens;
  const int* table;
  const float* ks;
  const float* vs;
  float* scratch;                               // [rows][heads][splits][hd + 2] where a row's pages are dealt out to several blocks
  int table_width, n_seqs, n_heads, kv_heads, hd, window, keep_first, splits, split_pages, skip_copy;
  float scale_log2;
};

// HDP: entries of a head, rounded up to a power of two; the rest come as zeros.
template <int HDP, int PIECES> struct Layout {
  static constexpr int PITCH = HDP < 128 ? HDP : 128, BLOCKS = (HDP + 127) / 128;      // bytes of a swizzled row; of them a key has so many
  static constexpr int KS = HDP / 16;                            // 16-entry steps
  static constexpr uint32_t TILE = PAGE * HDP;
  static constexpr uint32_t WARP = 2 * TILE + 2 * PAGE * 4;      // keys, values, their scales
  static constexpr uint32_t OFF_Q = 1024;                        // (mbarriers and the like before)
  static constexpr uint32_t Q_BYTES = PIECES * KS * 512;
  static constexpr uint32_t OFF_WARPS = (OFF_Q + Q_BYTES + 1023) / 1024 * 1024;
  static constexpr size_t smem(int warps) { return OFF_WARPS + (size_t)warps * ((WARP + 1023) / 1024 * 1024) + 1024; }
};

__device__ __forceinline__ uint32_t as_bits(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float power_of_2(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }
__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// Two of a word's four codes as half precision; SEL says which.
template <uint32_t SEL> __device__ __forceinline__ uint32_t two_codes(uint32_t offset_word) {
  return as_bits(__hsub2(as_half2(__byte_perm(offset_word, 0x64646464u, SEL)), as_half2(0x64806480u)));
}
// Where 16-byte piece c of a page's row lies: swizzled by TMA within spans of the row's length.
template <int HDP> __device__ __forceinline__ uint32_t place(int row, int c) {
  if (HDP == 16) return row * 16;
  if (HDP == 32) return row * 32 + ((c ^ ((row >> 2) & 1)) << 4);
  if (HDP == 64) return row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
  return (c >> 3) * (PAGE * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
}

template <typename T, int HDP>
__global__ void __launch_bounds__(256)
attention_int8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Args a) {
  constexpr int PIECES = std::is_same<T, float>::value ? 2 : 1;
  using L = Layout<HDP, PIECES>;
  constexpr int KS = L::KS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warps = blockDim.x >> 5;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem) + 2 * warp;                    // a page's keys, its values have come
  volatile int* failed = reinterpret_cast<volatile int*>(smem + 256);
  float* row_mul = reinterpret_cast<float*>(smem + 512);                           // [ROWS] what the queries were divided by
  uint4* q_frag = reinterpret_cast<uint4*>(smem + L::OFF_Q);                       // [piece][step][lane]
  uint8_t* mine = smem + L::OFF_WARPS + warp * ((L::WARP + 1023) / 1024 * 1024);
  uint8_t* k_tile = mine;
  uint8_t* v_tile = mine + L::TILE;
  float* ks = reinterpret_cast<float*>(mine + 2 * L::TILE);
  float* vs = ks + PAGE;

  pdl_launch_dependents();
  const int group = a.n_heads / a.kv_heads, heads = min(group, ROWS), tok = ROWS / heads, chunks = (group + heads - 1) / heads;
  // block: from the last tile of rows (which sees the most) on, then sequences and heads; a range of pages of them
  const int columns = a.n_seqs * a.kv_heads * chunks, split = blockIdx.y;
  const int from_end = blockIdx.x / columns;
  int rest = blockIdx.x - from_end * columns;
  const int s = rest / (a.kv_heads * chunks);
  rest -= s * a.kv_heads * chunks;
  const int kvh = rest / chunks, h0 = kvh * group + (rest - kvh * chunks) * heads, n_heads = min(heads, (kvh + 1) * group - h0);
  pdl_wait();
  const int row0 = a.seq_starts[s], n_new = a.seq_starts[s + 1] - row0;
  const int tile = (n_new + tok - 1) / tok - 1 - from_end;
  if (tile < 0) return;
  const int kv_len = a.kv_lens[s], n_tok = min(tok, n_new - tile * tok);
  const int pos0 = kv_len - n_new + tile * tok, last_pos = pos0 + n_tok - 1;
  const int first_page = a.window > 0 ? max(0, pos0 - a.window + 1) / PAGE : 0;
  const int kept = min((a.keep_first + PAGE - 1) / PAGE, first_page);
  const int units = kept + last_pos / PAGE - first_page + 1;
  auto page_of = [&](int u) { return u < kept ? u : first_page + u - kept; };
  const int u_begin = split * a.split_pages, u_end = a.splits > 1 ? min(units, u_begin + a.split_pages) : units;
  const int* pages = a.table + (int64_t)s * a.table_width;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
    *failed = 0;
  }
  if (lane == 0) {
    mbar_init(&bars[0], 1);
    mbar_init(&bars[1], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncwarp();

  // a lane has the number of every 32nd page of this warp's
  int u = u_begin + warp, ahead = 0, id = 0;
  auto ids = [&](int from) { id = from + lane * warps < u_end ? pages[page_of(from + lane * warps)] : 0; };
  ids(u);
  auto ask = [&](bool values, int64_t page, bool skip) {         // (lane 0)
    uint64_t* bar = &bars[values ? 1 : 0];
    const int64_t cell = (page * a.kv_heads + kvh) * PAGE;
    uint8_t* dst = values ? v_tile : k_tile;
    mbar_expect_tx(bar, L::TILE + PAGE * 4);
    if (!skip)
      for (int b = 0; b < L::BLOCKS; ++b) tma_load_2d(dst + b * PAGE * 128, values ? &map_v : &map_k, bar, b * 128, (int)cell);
    bulk_copy(values ? vs : ks, (values ? a.vs : a.ks) + cell, PAGE * 4, bar);
  };
  const int first_id = __shfl_sync(0xffffffffu, id, 0);
  if (lane == 0 && u < u_end) {
    ask(false, first_id, a.skip_copy);
    ask(true, first_id, false);
  }

  // the rows' queries: a warp takes rows one after another, a lane every 32nd entry; their largest exponent, then pieces where the products want them
  for (int r = warp; r < ROWS; r += warps) {
    const int token = r / heads, head = r - token * heads;
    const bool there = token < n_tok && head < n_heads;
    const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(row0 + tile * tok + token) * a.ld_q + (int64_t)(h0 + head) * a.hd;
    float x[(HDP + 31) / 32];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < (HDP + 31) / 32; ++i) {
      const int d = i * 32 + lane;
      x[i] = there && d < a.hd ? to_f32(src[d]) : 0.f;
      top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    }
    const uint32_t e = __reduce_max_sync(0xffffffffu, top) >> 23, used = e == 255 ? 127u : min(max(e, 1u), 253u);      // (a row that is not finite stays so)
    const float f = __uint_as_float((254u - used) << 23);
    if (lane == 0) row_mul[r] = __uint_as_float(used << 23);
#pragma unroll
    for (int i = 0; i < (HDP + 31) / 32; ++i) {
      const int d = i * 32 + lane, step = d >> 4, tt = (d >> 2) & 3, e4 = d & 3;      // entry of step `step`: thread tt's, the e4-th of its four
      if (d < HDP) {
        float y = x[i] * f;
        const int reg = (e4 >> 1) * 2 + (r >> 3);                // a0, a1: entries 0 and 1 of rows g and g + 8; a2, a3: entries 2 and 3
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
          const __half h = __float2half_rn(y);
          reinterpret_cast<__half*>(q_frag)[((size_t)(p * KS + step) * 32 + (r & 7) * 4 + tt) * 8 + reg * 2 + (e4 & 1)] = h;
          y -= __half2float(h);
        }
      }
    }
  }
  __syncthreads();

  float o[2 * KS][4];
#pragma unroll
  for (int i = 0; i < 2 * KS; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float ref[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};    // of rows g and g + 8; sums of this thread's keys
  const int pos[2] = {pos0 + g / heads, pos0 + (g + 8) / heads};
  const float mul[2] = {row_mul[g] * a.scale_log2, row_mul[g + 8] * a.scale_log2};
  int exponent = -64;
  uint32_t phase = 0;
  bool ok = true;
  const uint32_t k_addr = smem_u32(k_tile), v_addr = smem_u32(v_tile);

  for (; u < u_end; u += warps, phase ^= 1) {
    if (++ahead == 32) {
      ahead = 0;
      ids(u + warps);
    }
    const int next_id = __shfl_sync(0xffffffffu, id, ahead);
    const bool more = u + warps < u_end;
    const int page = page_of(u), there = kv_len - page * PAGE;
    // ---- scores: 16 rows x 64 keys
    if (!mbar_wait(&bars[0], phase)) { ok = false; break; }
    float sc[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
    constexpr int STEPS = KS < 4 ? KS : 4, TILES = 4 / STEPS;    // four matrices a load: so many steps of so many groups of eight keys
#pragma unroll
    for (int s0 = 0; s0 < KS; s0 += STEPS) {
      uint4 qf[PIECES][STEPS];
#pragma unroll
      for (int p = 0; p < PIECES; ++p)
#pragma unroll
        for (int i = 0; i < STEPS; ++i) qf[p][i] = q_frag[(p * KS + s0 + i) * 32 + lane];
#pragma unroll
      for (int n = 0; n < 8; n += TILES) {
        uint32_t w[4];
        const int m = lane >> 3;                                 // the matrix whose row this lane points at
        ldmatrix4(k_addr + place<HDP>((n + m / STEPS) * 8 + (lane & 7), s0 + m % STEPS), w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t x = w[i] ^ 0x80808080u, b0 = two_codes<0x4140>(x), b1 = two_codes<0x4342>(x);
#pragma unroll
          for (int p = PIECES - 1; p >= 0; --p) mma_f16(sc[n + i / STEPS], qf[p][i % STEPS], b0, b1);
        }
      }
    }
    // scores in powers of two
    float scale[8][2];
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const float2 k2 = *reinterpret_cast<const float2*>(ks + n * 8 + 2 * t);
      scale[n][0] = k2.x;
      scale[n][1] = k2.y;
    }
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[n][e] *= scale[n][e & 1] * mul[e >> 1];
    __syncwarp();
    if (lane == 0 && more) ask(false, next_id, false);           // these keys have been read
    const bool masked = page * PAGE + PAGE - 1 > pos0 || (a.window > 0 && page * PAGE <= last_pos - a.window && page * PAGE + PAGE > a.keep_first);
    if (masked) {
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = page * PAGE + n * 8 + 2 * t + (e & 1), p = pos[e >> 1];
          if (!(key <= p && (a.window == 0 || p - key < a.window || key < a.keep_first))) sc[n][e] = -INFINITY;
        }
    }
    // ---- weights
    if (!mbar_wait(&bars[1], phase)) { ok = false; break; }
    float vsc[8][2];
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const float2 v2 = *reinterpret_cast<const float2*>(vs + n * 8 + 2 * t);
      vsc[n][0] = v2.x;
      vsc[n][1] = v2.y;
    }
    {
      uint32_t top = 0;                                          // the exponent of the largest of the page's scales that is finite and the sequence's
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t bits = __float_as_uint(vsc[n][e]) & 0x7fffffffu;
          if (n * 8 + 2 * t + e < there && bits < 0x7f800000u) top = max(top, bits);
        }
      top = __reduce_max_sync(0xffffffffu, top) >> 23;
      if (top > 0) exponent = (int)top - 127;                    // (a page of zeros takes that of the values before)
    }
    const float c = (float)exponent, down = power_of_2(-exponent);
    float keep[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float m = -INFINITY;
#pragma unroll
      for (int n = 0; n < 8; ++n) m = fmaxf(m, fmaxf(sc[n][2 * r], sc[n][2 * r + 1]));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2)) + c;
      const float to = fmaxf(ref[r], m);
      keep[r] = to == -INFINITY ? 1.f : exp2_fast(ref[r] - to);
      ref[r] = to;
      const float add = c + HEAD - (to == -INFINITY ? 0.f : to);
      float part = 0.f;
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = exp2_fast(sc[n][2 * r + e] + add);
          part += p;
          const float w = p * (vsc[n][e] * down);
          sc[n][2 * r + e] = masked && sc[n][2 * r + e] == -INFINITY ? 0.f : w;      // (a scale that is not finite is for those alone who see it)
        }
      sum[r] = fmaf(sum[r], keep[r], part * down);
    }
    // ---- outputs: 64 keys x HDP.  In 32-bit a page's products have an accumulator of their own that joins the running output by a rounded addition: the tensor core
    // truncates what it adds up, which over a long sequence would show.
    constexpr bool APART = PIECES == 2;
    if (!APART && __any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] *= keep[e >> 1];
    }
    uint4 pf[PIECES][4];                                         // of 16 keys each
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {                              // a0, a1: eight keys of rows g and g + 8; a2, a3: the next eight
        float x = sc[2 * j + (i >> 1)][(i & 1) * 2], y = sc[2 * j + (i >> 1)][(i & 1) * 2 + 1];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
          const __half2 h = __floats2half2_rn(x, y);
          (i == 0 ? pf[p][j].x : i == 1 ? pf[p][j].y : i == 2 ? pf[p][j].z : pf[p][j].w) = as_bits(h);
          x -= __low2float(h);
          y -= __high2float(h);
        }
      }
#pragma unroll
    for (int c0 = 0; c0 < KS; c0 += 2) {                         // two pieces of 16 entries (one where a head has no more)
      constexpr int NC = KS == 1 ? 1 : 2;
      float fresh[2 * NC][4];
#pragma unroll
      for (int i = 0; i < 2 * NC; ++i) fresh[i][0] = fresh[i][1] = fresh[i][2] = fresh[i][3] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t w[4];
        const int m = lane >> 3, col = KS == 1 ? 0 : c0 + (m >> 1);
        ldmatrix4_trans(v_addr + place<HDP>(j * 16 + (m & 1) * 8 + (lane & 7), col), w);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const uint32_t x = w[2 * i] ^ 0x80808080u, y = w[2 * i + 1] ^ 0x80808080u;
          const uint32_t e0 = two_codes<0x4240>(x), e1 = two_codes<0x4240>(y), d0 = two_codes<0x4341>(x), d1 = two_codes<0x4341>(y);
#pragma unroll
          for (int p = PIECES - 1; p >= 0; --p) {
            mma_f16(APART ? fresh[2 * i] : o[2 * (c0 + i)], pf[p][j], e0, e1);                      // entries 2g of the sixteen
            mma_f16(APART ? fresh[2 * i + 1] : o[2 * (c0 + i) + 1], pf[p][j], d0, d1);              // entries 2g + 1
          }
        }
      }
      if (APART) {
#pragma unroll
        for (int i = 0; i < 2 * NC; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[2 * c0 + i][e] = fmaf(o[2 * c0 + i][e], keep[e >> 1], fresh[i][e]);
      }
    }
    __syncwarp();
    if (lane == 0 && more) ask(true, next_id, false);            // these values have been read
  }
  if (!ok) *failed = 1;

  // ---- the warps meet: outputs in the keys' place, maxima and sums in the scales'
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
  }
  const bool worked = u_begin + warp < u_end;
  if (worked && ok) {
    float4* dst = reinterpret_cast<float4*>(k_tile);             // [ROWS][HDP], four entries at a time, turned by the row against bank conflicts
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r)                                // entries 16 i + 4 t ..: 2 (2t) + {0, 1}, 2 (2t + 1) + {0, 1}
        dst[(g + 8 * r) * (HDP / 4) + ((4 * i + t) ^ (g & (HDP / 4 < 8 ? HDP / 4 - 1 : 7)))] =
            make_float4(o[2 * i][2 * r], o[2 * i + 1][2 * r], o[2 * i][2 * r + 1], o[2 * i + 1][2 * r + 1]);
  }
  if (t == 0) {
    ks[g] = worked ? ref[0] : -INFINITY;
    ks[g + 8] = worked ? ref[1] : -INFINITY;
    vs[g] = sum[0];
    vs[g + 8] = sum[1];
  }
  __syncthreads();
  if (*failed) {
    outlast_what_is_in_flight();
    return;
  }
  const int busy = max(0, min(warps, u_end - u_begin));
  const size_t stride = (L::WARP + 1023) / 1024 * 1024;
  const uint8_t* base = smem + L::OFF_WARPS;
  for (int i = threadIdx.x; i < ROWS * (HDP / 4); i += blockDim.x) {
    const int r = i / (HDP / 4), d4 = i - r * (HDP / 4), token = r / heads, head = r - token * heads;
    if (token >= n_tok || head >= n_heads || d4 * 4 >= a.hd) continue;
    float top = -INFINITY, l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < busy; ++w) top = fmaxf(top, reinterpret_cast<const float*>(base + w * stride + 2 * L::TILE)[r]);
    for (int w = 0; w < busy; ++w) {
      const float* m = reinterpret_cast<const float*>(base + w * stride + 2 * L::TILE);
      const float f = m[r] == -INFINITY ? 0.f : exp2_fast(m[r] - top);
      const float4 y = reinterpret_cast<const float4*>(base + w * stride)[r * (HDP / 4) + (d4 ^ (r & (HDP / 4 < 8 ? HDP / 4 - 1 : 7)))];
      l = fmaf(m[PAGE + r], f, l);
      x.x = fmaf(y.x, f, x.x); x.y = fmaf(y.y, f, x.y); x.z = fmaf(y.z, f, x.z); x.w = fmaf(y.w, f, x.w);
    }
    const int64_t row = row0 + tile * tok + token;
    if (a.splits > 1) {
      float* dst = a.scratch + ((row * a.n_heads + h0 + head) * a.splits + split) * (a.hd + 2);
      if (d4 == 0) dst[a.hd] = top, dst[a.hd + 1] = l;
      if (busy > 0) dst[d4 * 4] = x.x, dst[d4 * 4 + 1] = x.y, dst[d4 * 4 + 2] = x.z, dst[d4 * 4 + 3] = x.w;
    } else {
      T* dst = reinterpret_cast<T*>(a.out) + row * a.ld_out + (int64_t)(h0 + head) * a.hd + d4 * 4;
      const float inv = 1.f / l;
      dst[0] = from_f32<T>(x.x * inv); dst[1] = from_f32<T>(x.y * inv); dst[2] = from_f32<T>(x.z * inv); dst[3] = from_f32<T>(x.w * inv);
    }
  }
}

// The blocks of a row and head meet: a warp for each.
template <typename T>
__global__ void __launch_bounds__(128)
attention_int8_join_kernel(const float* __restrict__ scratch, T* __restrict__ out, int64_t ld_out, int n_rows, int n_heads, int hd, int splits) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_wait();
  if (item >= (int64_t)n_rows * n_heads) return;
  const float* src = scratch + item * splits * (hd + 2);
  float top = -INFINITY;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, src[s * (hd + 2) + hd]);
  float x[8] = {}, l = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float m = src[s * (hd + 2) + hd];
    if (m == -INFINITY) continue;                                // (a block without pages leaves no output)
    const float f = exp2_fast(m - top);
    l = fmaf(src[s * (hd + 2) + hd + 1], f, l);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * 32 + lane < hd) x[i] = fmaf(src[s * (hd + 2) + i * 32 + lane], f, x[i]);
  }
  const int64_t row = item / n_heads;
  T* dst = out + row * ld_out + (item - row * n_heads) * hd;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i * 32 + lane < hd) dst[i * 32 + lane] = from_f32<T>(x[i] / l);
}

// [rows of all pages][hd] bytes, a page's rows a copy.
int tensor_map(const int8_t* p, int64_t rows, int hd, int pitch, CUtensorMap* map) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) KVAD_FAIL(KVAD_ERR_CUDA, "attention_int8: the driver does not offer cuTensorMapEncodeTiled");
  cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)hd};
  cuuint32_t box[2] = {(cuuint32_t)pitch, PAGE}, elem[2] = {1, 1};
  const CUtensorMapSwizzle swizzle = pitch == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : pitch == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                     : pitch == 32 ? CU_TENSOR_MAP_SWIZZLE_32B : CU_TENSOR_MAP_SWIZZLE_NONE;
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(p), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) KVAD_FAIL(KVAD_ERR_CUDA, "attention_int8: cuTensorMapEncodeTiled failed (%d) for %lld rows of %d", (int)r, (long long)rows, hd);
  return KVAD_OK;
}

template <typename T, int HDP>
int launch(const Args& a, const int8_t* k, const int8_t* v, int64_t cache_rows, int max_new, int warps, cudaStream_t stream) {
  constexpr int PIECES = std::is_same<T, float>::value ? 2 : 1;
  using L = Layout<HDP, PIECES>;
  CUtensorMap mk, mv;
  int rc = tensor_map(k, cache_rows, a.hd, L::PITCH, &mk);
  if (rc == KVAD_OK) rc = tensor_map(v, cache_rows, a.hd, L::PITCH, &mv);
  if (rc != KVAD_OK) return rc;
  auto kernel = attention_int8_kernel<T, HDP>;
  while (warps > 1 && L::smem(warps) > 227 * 1024) warps /= 2;
  static bool configured = false;
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) KVAD_FAIL(KVAD_ERR_CUDA, "attention_int8: cannot reserve shared memory: %s", cudaGetErrorString(e));
    configured = true;
  }
  const int group = a.n_heads / a.kv_heads, heads = group < ROWS ? group : ROWS, tok = ROWS / heads, chunks = (group + heads - 1) / heads;
  const int64_t blocks = (int64_t)((max_new + tok - 1) / tok) * a.n_seqs * a.kv_heads * chunks;
  KVAD_REQUIRE(blocks < (1ll << 31) && a.splits <= 65535, "attention_int8: more rows and heads than a launch takes");
  const cudaError_t e = kvad_launch(kernel, dim3((unsigned)blocks, a.splits), dim3(warps * 32), L::smem(warps), stream, mk, mv, a);
  if (e != cudaSuccess) KVAD_FAIL(KVAD_ERR_CUDA, "attention_int8: launch failed: %s", cudaGetErrorString(e));
  return KVAD_OK;
}

template <typename T>
int by_size(const Args& a, const int8_t* k, const int8_t* v, int64_t cache_rows, int n_rows, int max_new, int warps, cudaStream_t stream) {
  const int rc = a.hd <= 16 ? launch<T, 16>(a, k, v, cache_rows, max_new, warps, stream) : a.hd <= 32 ? launch<T, 32>(a, k, v, cache_rows, max_new, warps, stream)
                 : a.hd <= 64 ? launch<T, 64>(a, k, v, cache_rows, max_new, warps, stream) : a.hd <= 128 ? launch<T, 128>(a, k, v, cache_rows, max_new, warps, stream)
                                                                                             : launch<T, 256>(a, k, v, cache_rows, max_new, warps, stream);
  if (rc != KVAD_OK || a.splits == 1) return rc;
  const int64_t blocks = ((int64_t)n_rows * a.n_heads + 3) / 4;
  KVAD_REQUIRE(blocks < (1ll << 31), "attention_int8: more rows and heads than a launch takes");
  const cudaError_t e = kvad_launch(attention_int8_join_kernel<T>, dim3((unsigned)blocks), dim3(128), 0, stream, (const float*)a.scratch,
                                    reinterpret_cast<T*>(a.out), a.ld_out, n_rows, a.n_heads, a.hd, a.splits);
  if (e != cudaSuccess) KVAD_FAIL(KVAD_ERR_CUDA, "attention_int8: launch failed: %s", cudaGetErrorString(e));
  return KVAD_OK;
}

}  // namespace

// `splits` > 1: the pages that a row sees are dealt out to that many blocks, `split_pages` each, through `scratch` (float32, rows x heads x splits x (head size + 2));
// `warps`: of a block, 4 or 8 (fewer where a head's pages are too large).
KVAD_EXPORT int kvad_attention_int8(int dtype, const void* q, int64_t ld_q, void* out, int64_t ld_o, const int* seq_starts, const int* kv_lens,
                                    const int* table, int table_width, const int8_t* k_pages, const float* k_scales, const int8_t* v_pages,
                                    const float* v_scales, int n_pages, int n_rows, int n_seqs, int max_new, int n_heads, int kv_heads, int hd, int page,
                                    float scale, int window, int keep_first, int splits, int split_pages, int warps, void* scratch, cudaStream_t stream) {
  KVAD_REQUIRE(n_rows > 0 && n_seqs > 0 && max_new > 0 && table_width > 0 && n_pages > 0, "attention_int8: needs rows, sequences and pages");
  KVAD_REQUIRE(n_heads > 0 && kv_heads > 0 && n_heads % kv_heads == 0, "attention_int8: %d heads do not divide into %d key/value heads", n_heads, kv_heads);
  if (hd <= 0 || hd % 16 || hd > 256) KVAD_FAIL(KVAD_ERR_UNSUPPORTED, "attention_int8: head sizes are multiples of 16 up to 256, not %d", hd);
  if (page != PAGE) KVAD_FAIL(KVAD_ERR_UNSUPPORTED, "attention_int8: pages hold 64 positions, not %d", page);
  KVAD_REQUIRE(((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) | reinterpret_cast<uintptr_t>(k_scales) |
                 reinterpret_cast<uintptr_t>(v_scales)) & 15) == 0, "attention_int8: pages and scales must start on a 16-byte boundary");
  KVAD_REQUIRE(window >= 0 && keep_first >= 0, "attention_int8: a window and kept first positions cannot be negative");
  KVAD_REQUIRE(warps >= 1 && warps <= 8 && splits >= 1 && (splits == 1 || (split_pages > 0 && scratch != nullptr)), "attention_int8: no way to deal out pages: %d, %d, %d",
               splits, split_pages, warps);
  const int64_t cache_rows = (int64_t)n_pages * kv_heads * PAGE;
  KVAD_REQUIRE(cache_rows < (1ll << 31), "attention_int8: more cached rows than a copy can name");
  const Args a{q, ld_q, out, ld_o, seq_starts, kv_lens, table, k_scales, v_scales, reinterpret_cast<float*>(scratch), table_width, n_seqs, n_heads, kv_heads, hd,
               window, window > 0 ? keep_first : 0, splits, split_pages, g_skip_copy ? 1 : 0, scale * LOG2E};
  g_skip_copy = false;
  const int rc = dtype == KVAD_DTYPE_F32 ? by_size<float>(a, k_pages, v_pages, cache_rows, n_rows, max_new, warps, stream)
                                         : by_size<__nv_bfloat16>(a, k_pages, v_pages, cache_rows, n_rows, max_new, warps, stream);
  if (rc != KVAD_OK) return rc;
  KVAD_CHECK_LAUNCH("attention_int8");
  return KVAD_OK;
}

// How many bounded waits have run out in this process (0 unless something is wrong).  Synchronises the device.
KVAD_EXPORT int kvad_attention_int8_status() {
  int n = 0;
  if (cudaMemcpyFromSymbol(&n, g_wait_timeouts, sizeof(n)) != cudaSuccess) return -1;
  return n;
}

// Tests of the bounded waits: `wait_limit` > 0 sets how many polls a wait makes before it gives up (0: the library's own limit); `skip_copy` leaves the first
// page's keys out of the NEXT launch's warps, so that the wait for them runs out.  Synchronises the device.
KVAD_EXPORT int kvad_attention_int8_test_hooks(unsigned wait_limit, int skip_copy) {
  g_skip_copy = skip_copy;
  return set_wait_limit(wait_limit);
}
