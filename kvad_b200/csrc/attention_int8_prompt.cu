// Causal attention of prompt rows over the paged cache of 8-bit codes, on the 5th-generation tensor cores (bfloat16, heads of up to 128 entries).
//
//   t_ij = log2(e) scale ks_j (q_i . kc_j) + log2(vs_j),    p_ij = 2^(t_ij - m_i),    out_i = sum_j p_ij vc_j / sum_j p_ij / vs_j
//
// with kc, vc the codes of key and value j and ks, vs their scales: p is the softmax's weight times the value's scale.  Codes are whole numbers of -127 .. 127, which
// bfloat16 holds exactly, so both products take the codes as they are and the scales come in as three numbers a key, one multiply-add on the score and one in the sum.
// What is rounded to bfloat16 is p, as the second product's operand, and the output; scores, maxima, sums and outputs are 32-bit.  With the value's scale inside the exponent the
// largest p of a row is a power of two, so that a row that attends to one key has that key's value as it is kept.  (A value's scale below 2^-100 counts as 2^-100:
// weights of keys whose scales are less than 2^100 apart stay within 32-bit numbers.)
//
// A block has two SLOTS of 128 rows: rows are (token, head) pairs of one key/value head's group, so that the heads that share keys share the work of bringing them.
// Keys come in steps of two pages (128).  Roles, by warp:
//   0       brings the queries by TMA and the pages' codes and scales, as they lie, by bulk copies into a ring
//   1, 2    issue the products of a slot each:  S = Q K^T (128 x 128), then T += P V with P in tensor memory, over S's own columns
//   4-7     turn codes to bfloat16 in the layout the products read (128-byte swizzle): two shifts of bytes to a place, two masks and one subtraction for two
//           entries, once for both slots' 256 rows
//   8-11, 12-15  a thread a row: scores to weights.  The running output stays in tensor memory; it is scaled down only when a row's maximum has risen by
//           more than 2^8 since the last time (weights are then at most 2^8, and as exact as any), which after the first steps is hardly ever
//
// Keys a row does not see weigh nothing; what a page holds beyond the sequence's end are some codes, which are finite, with scales that are not looked at.
// Every wait is bounded; one that runs out raises a counter and the block frees its tensor memory and returns without writing.
#include "scored_tiles.cuh"

using namespace kvad;

KVAD_DEFINE_LAST_ERROR()

namespace {

constexpr int KEYS = 128;                       // of a step: two pages
constexpr int THREADS = 512;
constexpr int REGS_FEW = 56, REGS_TURN = 88, REGS_MANY = 184;       // of 128 a thread at launch: 56 + 88 + 2 * 184 = 4 * 128
constexpr int SCALE_SETS = 4;
constexpr float RISE = 8.f, LEAST = 0x1p-100f;

bool g_skip_copy = false;                       // tests: the next launch's blocks leave out their first page

struct Args {
  __nv_bfloat16* out;
  int64_t ld_out;
  const int* seq_starts;
  const int* kv_lens;
  const int* table;
  int table_width;
  const int8_t* k;
  const float* ks;
  const int8_t* v;
  const float* vs;
  int n_seqs, n_heads, kv_heads, window, keep_first, skip_copy;
  float scale_log2;
};

template <int HD> struct Layout {
  static constexpr int BLOCKS = (HD + 63) / 64;                  // of 64 entries: 128 bytes of bfloat16
  static constexpr int RING = HD > 64 ? 3 : 6, RAW = 6;         // keys or values of a step as bfloat16; of a page as they came
  static constexpr uint32_t BLOCK = 128 * 128;                   // 128 rows (or keys) of a block of entries
  static constexpr uint32_t Q_BYTES = BLOCKS * BLOCK, KV_BYTES = BLOCKS * BLOCK;
  static constexpr uint32_t CODES = PAGE * HD, RAW_BYTES = CODES + 2 * PAGE * 4;
  static constexpr uint32_t OFF_KV = 2 * Q_BYTES, OFF_RAW = OFF_KV + RING * KV_BYTES, OFF_SC = OFF_RAW + RAW * RAW_BYTES;
  static constexpr uint32_t OFF_BAR = OFF_SC + SCALE_SETS * 3 * KEYS * 4;
  static constexpr int BARS = 1 + 2 * RING + 2 * RAW + 2 * 3;
  static constexpr size_t SMEM = OFF_BAR + BARS * 8 + 16 + 1024;
  static constexpr uint32_t TM_O = 2 * KEYS;                     // S (and P) of slot t at t * 128, its output at TM_O + t * 128
  static_assert(SMEM <= 227 * 1024, "an SM's shared memory");
};

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void halves(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
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
__device__ __forceinline__ void scale_pair(uint32_t* x, uint64_t f, uint64_t g) {
  float u, v;
  halves(fma2(pair(__uint_as_float(x[0]), __uint_as_float(x[1])), f, g), u, v);
  x[0] = __float_as_uint(u);
  x[1] = __float_as_uint(v);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two codes, in bytes 0 and 2 of x, as bfloat16: 0x4300 is 128 and has room for seven bits, so 0x4300 | low seven bits is 128 + those, and what is to be
// taken off is 128, or 256 (0x4380) where the code's sign bit says that it stands for 128 less.
__device__ __forceinline__ uint32_t codes_to_bf16(uint32_t x) {
  const uint32_t a = (x & 0x007f007fu) | 0x43004300u, b = (x & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint64_t v_descriptor(uint32_t smem_addr, uint32_t block) {      // keys are the product's K, 128 contiguous bytes are 64 of its columns
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | (uint64_t)(block >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

template <int HD>
__global__ void __launch_bounds__(THREADS, 1)
attention_int8_prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ Args a) {
  using L = Layout<HD>;
  constexpr int RING = L::RING, RAW = L::RAW;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* q_tiles = smem;
  uint8_t* kv_tiles = smem + L::OFF_KV;
  uint8_t* raw_tiles = smem + L::OFF_RAW;
  float* scales = reinterpret_cast<float*>(smem + L::OFF_SC);   // [SCALE_SETS][keys' (times scale and log2 e), logarithms of values', values' inverses][128]
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* kv_full = q_full + 1;                                // [RING] keys or values of a step are bfloat16
  uint64_t* kv_empty = kv_full + RING;                           // [RING] both slots' products have read them
  uint64_t* raw_full = kv_empty + RING;                          // [RAW] a page's codes and scales have come
  uint64_t* raw_empty = raw_full + RAW;                          // [RAW] they have been turned
  uint64_t* s_full = raw_empty + RAW;                            // [slot] S is in tensor memory
  uint64_t* p_full = s_full + 2;                                 // [slot] P is (and S has been read)
  uint64_t* t_full = p_full + 2;                                 // [slot] P V has been added
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(t_full + 2);
  __shared__ int failed;

  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  const int group = a.n_heads / a.kv_heads, tok = ROWS / group;  // tokens of a slot
  const int columns = a.n_seqs * a.kv_heads, from_end = blockIdx.x / columns, column = blockIdx.x - from_end * columns;
  const int s = column / a.kv_heads, kvh = column - s * a.kv_heads;
  const int row0 = a.seq_starts[s], n_new = a.seq_starts[s + 1] - row0;
  const int tile = (n_new + 2 * tok - 1) / (2 * tok) - 1 - from_end;      // the last rows, which see the most, first
  if (tile < 0) return;
  const int kv_len = a.kv_lens[s];
  const int* pages = a.table + (int64_t)s * a.table_width;
  // this block's rows of each slot; the pages that any of them sees: the kept ones, then from first_page on
  const int tok0 = tile * 2 * tok, pos0 = kv_len - n_new + tok0;
  const int n_tok0 = min(tok, n_new - tok0), n_tok1 = max(0, min(tok, n_new - tok0 - tok));
  const int first_page = a.window > 0 ? max(0, pos0 - a.window + 1) / PAGE : 0;
  const int kept = min((a.keep_first + PAGE - 1) / PAGE, first_page);
  const int units0 = kept + (pos0 + n_tok0 - 1) / PAGE - first_page + 1;
  const int units1 = n_tok1 > 0 ? kept + (pos0 + tok + n_tok1 - 1) / PAGE - first_page + 1 : 0;
  const int units = max(units0, units1), steps = (units + 1) / 2;
  auto page_of = [&](int u) { return u < kept ? u : first_page + u - kept; };

  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_q);
    mbar_init(q_full, 1);
    for (int i = 0; i < RING; ++i) { mbar_init(&kv_full[i], 128); mbar_init(&kv_empty[i], 2); }
    for (int i = 0; i < RAW; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], 4); }
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 128); mbar_init(&t_full[i], 1); }
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_shared();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp < 4) {
    regs_fewer<REGS_FEW>();
    if (warp == 0) {
      if (lane == 0) {
        const uint32_t box = (uint32_t)(group * tok) * 128;
        mbar_expect_tx(q_full, (n_tok1 > 0 ? 2u : 1u) * L::BLOCKS * box);
        for (int t = 0; t < (n_tok1 > 0 ? 2 : 1); ++t)
          for (int b = 0; b < L::BLOCKS; ++b)
            tma_load_3d(q_tiles + t * L::Q_BYTES + b * L::BLOCK, &map_q, q_full, b * 64, kvh * group, row0 + tok0 + t * tok);
        int r = 0;
        uint32_t phase = 1;                                      // (the first round finds the ring empty)
        for (int u0 = 0; u0 < units && ok; u0 += 2) {
          for (int x = 0; x < 4; ++x) {                          // keys of two pages, then their values
            const int u = u0 + (x & 1);
            if (u >= units) continue;
            const int64_t cell = ((int64_t)pages[page_of(u)] * a.kv_heads + kvh) * PAGE;
            if (!mbar_wait(&raw_empty[r], phase)) { ok = false; break; }
            uint8_t* dst = raw_tiles + r * L::RAW_BYTES;
            mbar_expect_tx(&raw_full[r], L::CODES + (x < 2 ? 2 * PAGE * 4 : 0));
            if (!(a.skip_copy && u == 0 && x == 0)) bulk_copy(dst, (x < 2 ? a.k : a.v) + cell * HD, L::CODES, &raw_full[r]);
            if (x < 2) {                                         // both scales with the keys: scores want both
              bulk_copy(dst + L::CODES, a.ks + cell, PAGE * 4, &raw_full[r]);
              bulk_copy(dst + L::CODES + PAGE * 4, a.vs + cell, PAGE * 4, &raw_full[r]);
            }
            if (++r == RAW) r = 0, phase ^= 1;
          }
        }
      }
    } else if (warp < 3) {
      // ---- the products of a slot.  S of the next step goes over P, so it waits until P V has read it: meanwhile the tensor core works on the other slot
      const int t = warp - 1;
      const int mine = t == 0 ? (units0 + 1) / 2 : (units1 + 1) / 2;
      constexpr uint32_t idesc_s = umma_instr_desc(ROWS, KEYS), idesc_t = umma_instr_desc(ROWS, HD, false, true);
      const bool one = elect_one();
      const uint64_t q_desc = sw128_desc(smem_u32(q_tiles + t * L::Q_BYTES)), k_desc = sw128_desc(smem_u32(kv_tiles));
      const uint64_t v_desc = v_descriptor(smem_u32(kv_tiles), L::BLOCK);
      const uint32_t tm_s = tmem + t * KEYS, tm_o = tmem + L::TM_O + t * 128;
      int r = 0;
      uint32_t phase = 0;
      auto next = [&] { if (++r == RING) r = 0, phase ^= 1; };
      if (mine > 0) ok = mbar_wait(q_full, 0);
      for (int i = 0; i < steps && ok; ++i) {
        if (i < mine) {
          if (i > 0 && !mbar_wait(&t_full[t], (i - 1) & 1)) { ok = false; break; }
          if (!mbar_wait(&kv_full[r], phase)) { ok = false; break; }
          tc_fence_after();
          if (one) {
            const uint64_t at = k_desc + (uint32_t)r * (L::KV_BYTES >> 4);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
              const uint64_t off = (uint64_t)((k / 4) * (L::BLOCK >> 4) + (k % 4) * 2);
              umma(tm_s, q_desc + off, at + off, idesc_s, k > 0 ? 1u : 0u);
            }
            umma_commit(&s_full[t]);
            umma_commit(&kv_empty[r]);
          }
          next();
          if (!(mbar_wait(&p_full[t], i & 1) && mbar_wait(&kv_full[r], phase))) { ok = false; break; }
          tc_fence_after();
          if (one) {
            const uint64_t at = v_desc + (uint32_t)r * (L::KV_BYTES >> 4);
#pragma unroll
            for (int k = 0; k < KEYS / 16; ++k) umma_ta(tm_o, tm_s + k * 8, at + (uint64_t)(k * (2048 >> 4)), idesc_t, (i > 0 || k > 0) ? 1u : 0u);
            umma_commit(&t_full[t]);
            umma_commit(&kv_empty[r]);
          }
          next();
        } else {                                                 // the other slot walks on: give back what comes unread
          for (int x = 0; x < 2 && ok; ++x) {
            ok = mbar_wait(&kv_full[r], phase);
            if (ok && lane == 0) mbar_arrive_one(&kv_empty[r]);
            next();
          }
        }
      }
    }
  } else if (warp < 8) {
    // ---- codes to bfloat16
    regs_fewer<REGS_TURN>();
    const int tid = threadIdx.x - 128;
    int raw = 0, r = 0;
    uint32_t raw_phase = 0, phase = 1;
    for (int i = 0; i < steps && ok; ++i) {
      for (int x = 0; x < 2 && ok; ++x) {                        // keys, values
        if (!mbar_wait(&kv_empty[r], phase)) { ok = false; break; }
        uint8_t* dst = kv_tiles + r * L::KV_BYTES;
        float* sc = scales + (i % SCALE_SETS) * 3 * KEYS;
        for (int h = 0; h < 2; ++h) {                            // two pages
          const int u = 2 * i + h;
          if (u < units) {
            if (!mbar_wait(&raw_full[raw], raw_phase)) { ok = false; break; }
            const uint8_t* src = raw_tiles + raw * L::RAW_BYTES;
            constexpr int PER_ROW = HD / 16, PIECES = PAGE * PER_ROW;
            // a thread takes 16 codes; threads are dealt out so that eight neighbours read 128 bytes in a row and write pieces that lie in eight different banks' columns
#pragma unroll
            for (int p0 = 0; p0 < PIECES; p0 += 128) {
              const int p = p0 + tid;
              if (PIECES % 128 == 0 || p < PIECES) {
                int row, c;
                if (PER_ROW == 8) {
                  const int q = (p >> 2) & 3;
                  row = (p >> 4) * 2 + (q & 1);
                  c = (p & 3) + ((q == 1 || q == 2) ? 4 : 0);
                } else {
                  row = p / PER_ROW;
                  c = p - row * PER_ROW;
                }
                const int4 w = *reinterpret_cast<const int4*>(src + row * HD + c * 16);
                const uint32_t word[4] = {(uint32_t)w.x, (uint32_t)w.y, (uint32_t)w.z, (uint32_t)w.w};
                uint32_t e[8];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  e[2 * y] = codes_to_bf16(__byte_perm(word[y], 0, 0x4140));
                  e[2 * y + 1] = codes_to_bf16(__byte_perm(word[y], 0, 0x4342));
                }
                const int key = h * PAGE + row, piece = (c & 3) * 2;
                uint8_t* d = dst + (c >> 2) * L::BLOCK + key * 128;
                *reinterpret_cast<uint4*>(d + ((piece ^ (key & 7)) << 4)) = make_uint4(e[0], e[1], e[2], e[3]);
                *reinterpret_cast<uint4*>(d + (((piece + 1) ^ (key & 7)) << 4)) = make_uint4(e[4], e[5], e[6], e[7]);
              }
            }
            if (x == 0) {                                        // (beyond the sequence's end a scale may be anything)
              const int key = tid & (PAGE - 1);
              const bool there = page_of(u) * PAGE + key < kv_len;
              const float v = there ? reinterpret_cast<const float*>(src + L::CODES)[tid] : 1.f;
              if (tid < PAGE) {
                sc[h * PAGE + key] = v * a.scale_log2;
              } else {
                const float w = v < LEAST ? LEAST : v;           // (not a number stays what it is)
                sc[KEYS + h * PAGE + key] = log2f(w);
                sc[2 * KEYS + h * PAGE + key] = 1.f / w;
              }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive_one(&raw_empty[raw]);
            if (++raw == RAW) raw = 0, raw_phase ^= 1;
          } else {                                               // no second page: keys of zeros
            for (int p = tid; p < L::BLOCKS * PAGE * 8; p += 128)
              *reinterpret_cast<uint4*>(dst + (p / (PAGE * 8)) * L::BLOCK + PAGE * 128 + (p % (PAGE * 8)) * 16) = make_uint4(0, 0, 0, 0);
            if (x == 0 && tid < PAGE) sc[PAGE + tid] = sc[KEYS + PAGE + tid] = sc[2 * KEYS + PAGE + tid] = 1.f;
          }
        }
        if (!ok) break;
        fence_async_shared();
        mbar_arrive_one(&kv_full[r]);
        if (++r == RING) r = 0, phase ^= 1;
      }
    }
  } else {
    // ---- scores to weights: a thread a row
    regs_more<REGS_MANY>();
    const int t = (warp - 8) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const int mine = t == 0 ? (units0 + 1) / 2 : (units1 + 1) / 2, n_tok = t == 0 ? n_tok0 : n_tok1;
    const int first_pos = pos0 + t * tok, last_pos = first_pos + n_tok - 1, pos = first_pos + row / group;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t tm_s = tmem + t * KEYS + lanes, tm_o = tmem + L::TM_O + t * 128 + lanes;
    // whether every row of the slot sees every key of a page
    auto whole = [&](int page) {
      return page * PAGE + PAGE - 1 <= first_pos && (a.window == 0 || page * PAGE > last_pos - a.window || page * PAGE + PAGE <= a.keep_first);
    };
    float ref = -INFINITY;                       // what the weights are relative to: the row's maximum, or up to RISE less
    uint64_t sum[2] = {0, 0};
    for (int i = 0; i < mine; ++i) {
      const int page0 = page_of(2 * i), page1 = 2 * i + 1 < units ? page_of(2 * i + 1) : 1 << 24;      // (no second page: keys that nobody sees)
      const bool masked = !(whole(page0) && 2 * i + 1 < units && whole(page1));
      const float* ks = scales + (i % SCALE_SETS) * 3 * KEYS;
      const float* vl = ks + KEYS;
      const float* vi = vl + KEYS;
      if (!mbar_wait(&s_full[t], i & 1)) { ok = false; break; }
      tc_fence_after();
      uint32_t x[KEYS];                          // the row's scores, in place
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c0 = 0; c0 < KEYS; c0 += 32) tmem_ld32(tm_s + c0, x + c0);
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < KEYS; c += 4) {
        const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(ks + c), g = *reinterpret_cast<const ulonglong2*>(vl + c);
        scale_pair(x + c, f.x, g.x);
        scale_pair(x + c + 2, f.y, g.y);
      }
      if (masked) {
#pragma unroll
        for (int c = 0; c < KEYS; ++c) {
          const int key = (c < PAGE ? page0 * PAGE : page1 * PAGE - PAGE) + c;
          if (!(key <= pos && (a.window == 0 || pos - key < a.window || key < a.keep_first))) x[c] = 0xff800000u;
        }
      }
#pragma unroll
      for (int c = 0; c < KEYS; c += 2) top[(c >> 1) & 3] = fmaxf(top[(c >> 1) & 3], fmaxf(__uint_as_float(x[c]), __uint_as_float(x[c + 1])));
      const float peak = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      if (i == 0) {
        ref = peak;
      } else if (__any_sync(0xffffffffu, peak > ref + RISE)) {   // (S of this step was begun after P V of the last had ended: the output is at rest)
        const float to = fmaxf(ref, peak), keep = ref == -INFINITY ? 0.f : exp2_fast(ref - to);
        const uint64_t keep2 = pair(keep, keep);
        sum[0] = fma2(sum[0], keep2, 0);
        sum[1] = fma2(sum[1], keep2, 0);
        ref = to;
#pragma unroll
        for (int c0 = 0; c0 < HD; c0 += 16) {
          float o[16];
          tmem_ld16(tm_o + c0, o);
          uint32_t w[2][8];
#pragma unroll
          for (int c = 0; c < 16; ++c) w[c >> 3][c & 7] = __float_as_uint(o[c] * keep);
          tmem_st8(tm_o + c0, w[0]);
          tmem_st8(tm_o + c0 + 8, w[1]);
        }
      }
      const float base = ref == -INFINITY ? 0.f : -ref;          // a row that has seen nothing yet
      const uint64_t base2 = pair(base, base);
#pragma unroll
      for (int c0 = 0; c0 < KEYS; c0 += 16) {
        uint32_t w[8];
#pragma unroll
        for (int c = 0; c < 16; c += 4) {
          const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(vi + c0 + c);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float u = __uint_as_float(x[c0 + c + 2 * e]), v = __uint_as_float(x[c0 + c + 2 * e + 1]);
            float p, q;
            halves(add2(pair(u, v), base2), p, q);
            p = exp2_fast(p);
            q = exp2_fast(q);
            uint64_t g = e ? f.y : f.x;
            if (masked) {                                        // (a scale that is not finite is for those alone who see it)
              float y, z;
              halves(g, y, z);
              g = pair(u == -INFINITY ? 0.f : y, v == -INFINITY ? 0.f : z);
            }
            sum[e] = fma2(pair(p, q), g, sum[e]);
            w[c / 2 + e] = bf16_pair(p, q);
          }
        }
        tmem_st8(tm_s + c0 / 2, w);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive_one(&p_full[t]);
    }
    if (ok && mine > 0) {
      ok = mbar_wait(&t_full[t], (mine - 1) & 1);
      tc_fence_after();
      float u, v, u1, v1;
      halves(sum[0], u, v);
      halves(sum[1], u1, v1);
      const float inv = 1.f / ((u + v) + (u1 + v1));
      const int token = row / group, head = row - token * group;
      const bool there = ok && token < n_tok && !failed;
      __nv_bfloat16* dst = a.out + (int64_t)(row0 + tok0 + t * tok + token) * a.ld_out + (int64_t)(kvh * group + head) * HD;
#pragma unroll
      for (int c0 = 0; c0 < HD; c0 += 16) {
        float o[16];
        tmem_ld16(tm_o + c0, o);
        if (there) {
          uint32_t w[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) w[c] = bf16_pair(o[2 * c] * inv, o[2 * c + 1] * inv);
          *reinterpret_cast<uint4*>(dst + c0) = make_uint4(w[0], w[1], w[2], w[3]);
          *reinterpret_cast<uint4*>(dst + c0 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
        }
      }
    }
  }
  if (!ok) failed = 1;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (failed) outlast_what_is_in_flight();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD>
int launch(const void* q, int64_t ld_q, int n_rows, const Args& a, int max_new, cudaStream_t stream) {
  using L = Layout<HD>;
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) KVAD_FAIL(KVAD_ERR_CUDA, "attention_int8_prompt: the driver does not offer cuTensorMapEncodeTiled");
  const int group = a.n_heads / a.kv_heads, tok = ROWS / group;
  CUtensorMap map;
  cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)a.n_heads, (cuuint64_t)n_rows}, strides[2] = {HD * 2, (cuuint64_t)ld_q * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)tok}, elem[3] = {1, 1, 1};
  CUresult r = fn(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) KVAD_FAIL(KVAD_ERR_CUDA, "attention_int8_prompt: cuTensorMapEncodeTiled failed (%d) for %d rows, %lld apart", (int)r, n_rows, (long long)ld_q);
  auto kernel = attention_int8_prompt_kernel<HD>;
  static bool configured = false;
  if (!configured) {
    cudaFuncAttributes attr;
    cudaError_t e = cudaFuncGetAttributes(&attr, kernel);
    if (e == cudaSuccess && attr.numRegs != 65536 / THREADS)       // what the roles share out among themselves
      KVAD_FAIL(KVAD_ERR_CUDA, "attention_int8_prompt: built with %d registers a thread, not %d", attr.numRegs, 65536 / THREADS);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::SMEM);
    if (e != cudaSuccess) KVAD_FAIL(KVAD_ERR_CUDA, "attention_int8_prompt: cannot reserve %zu bytes of shared memory: %s", L::SMEM, cudaGetErrorString(e));
    configured = true;
  }
  const int64_t blocks = (int64_t)((max_new + 2 * tok - 1) / (2 * tok)) * a.n_seqs * a.kv_heads;
  KVAD_REQUIRE(blocks < (1ll << 31), "attention_int8_prompt: more rows and heads than a launch takes");
  const cudaError_t e = kvad_launch(kernel, dim3((unsigned)blocks), dim3(THREADS), L::SMEM, stream, map, a);
  if (e != cudaSuccess) KVAD_FAIL(KVAD_ERR_CUDA, "attention_int8_prompt: launch failed: %s", cudaGetErrorString(e));
  KVAD_CHECK_LAUNCH("attention_int8_prompt");
  return KVAD_OK;
}

}  // namespace

KVAD_EXPORT int kvad_attention_int8_prompt(const void* q, int64_t ld_q, void* out, int64_t ld_o, const int* seq_starts, const int* kv_lens, const int* table,
                                           int table_width, const int8_t* k_pages, const float* k_scales, const int8_t* v_pages, const float* v_scales, int n_rows,
                                           int n_seqs, int max_new, int n_heads, int kv_heads, int hd, int page, float scale, int window, int keep_first,
                                           cudaStream_t stream) {
  KVAD_REQUIRE(n_rows > 0 && n_seqs > 0 && max_new > 0 && table_width > 0, "attention_int8_prompt: needs rows, sequences and pages");
  KVAD_REQUIRE(n_heads > 0 && kv_heads > 0 && n_heads % kv_heads == 0, "attention_int8_prompt: %d heads do not divide into %d key/value heads", n_heads, kv_heads);
  KVAD_REQUIRE(page == PAGE, "attention_int8_prompt: pages hold 64 positions, not %d", page);
  KVAD_REQUIRE(n_heads / kv_heads <= ROWS, "attention_int8_prompt: at most 128 heads share a key/value head");
  KVAD_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) |
                 reinterpret_cast<uintptr_t>(k_scales) | reinterpret_cast<uintptr_t>(v_scales)) & 15) == 0 && ld_q % 8 == 0 && ld_o % 8 == 0,
               "attention_int8_prompt: rows, pages and scales must start on 16-byte boundaries");
  KVAD_REQUIRE(window >= 0 && keep_first >= 0, "attention_int8_prompt: a window and kept first positions cannot be negative");
  Args a{reinterpret_cast<__nv_bfloat16*>(out), ld_o, seq_starts, kv_lens, table, table_width, k_pages, k_scales, v_pages, v_scales,
         n_seqs, n_heads, kv_heads, window, window > 0 ? keep_first : 0, g_skip_copy ? 1 : 0, scale * LOG2E};
  g_skip_copy = false;
  switch (hd) {
    case 64: return launch<64>(q, ld_q, n_rows, a, max_new, stream);
    case 128: return launch<128>(q, ld_q, n_rows, a, max_new, stream);
    default: KVAD_FAIL(KVAD_ERR_UNSUPPORTED, "attention_int8_prompt: no kernel for heads of %d entries", hd);
  }
}

// How many bounded waits have run out in this process (0 unless something is wrong).  Synchronises the device.
KVAD_EXPORT int kvad_attention_int8_prompt_status() {
  int n = 0;
  if (cudaMemcpyFromSymbol(&n, g_wait_timeouts, sizeof(n)) != cudaSuccess) return -1;
  return n;
}

// Tests of the bounded waits: `wait_limit` > 0 sets how many polls a wait makes before it gives up (0: the library's own limit); `skip_copy` leaves the first
// page out of the NEXT launch's blocks, so that the wait for it runs out.  Synchronises the device.
KVAD_EXPORT int kvad_attention_int8_prompt_test_hooks(unsigned wait_limit, int skip_copy) {
  g_skip_copy = skip_copy;
  return set_wait_limit(wait_limit);
}
