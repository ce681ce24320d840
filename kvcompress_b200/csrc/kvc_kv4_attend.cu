// Attention over the pages of the 4-bit KV cache, for a few queries a KV head.
//
// For a query q and the tokens t of its sequence, o = sum_t p_t v_t / sum_t p_t
// with p_t = exp(scale q.k_t - m).  K and V are never dequantised: with k_t =
// z_t + s_t (c_t - 8) in each group,
//   q.k_t = s_t (q.c_t) + (z_t - 8 s_t) sum(q),
//   sum_t p_t v_t = sum_t (p_t s'_t) c'_t - 8 sum_t (p_t s'_t) + sum_t p_t z'_t,
// so the products run on the codes 0..15 themselves, as float16 operands of
// mma.sync m16n8k16 with float32 accumulators.  A nibble masked out of its word
// IS a float16: the bits 0x000n are the denormal n 2^-24 and 0x00n0 are
// n 2^-20, exactly, so a word of 8 codes becomes four operand registers with
// four ANDs and one shift.  The powers of two are taken out of the queries
// (every second operand register is met by q / 16) and out of the result.
//
// With float32 queries the codes are centred instead (c - 8 as float16 from
// 1024 + c, one more instruction a register): 8 s sum(q) and 8 s' are large
// against a logit and an average over many tokens, and the accumulators' own
// rounding would show (7e-6 of the result instead of 1e-6).  For the same
// reason they hold 16 tokens or features at most, and float32 additions join them.
//
// What the kernel rounds: queries of 16 bits not at all (float16 with a power
// of two per row), float32 ones to two float16 terms (22 bits); p s' to
// float16 under a power of two that keeps its maximum near the top of the
// range (two terms for float32 queries, the second under 2^11 more).  That power
// is each column's and group's own and goes by the tokens that the column sees, so
// that a quiet group beside a loud one, or queries before a loud token, keep their
// bits.  What remains: where p s' is below 2^-21 of its group's largest s' (p = 1 at
// the running maximum) it is rounded to steps of 2^-31 of that (2^-42 with two
// terms).  The sum that the constant 8 s' multiplies is formed from the rounded
// weights, so their rounding acts on c' - 8 and not on c'.
//
// A block takes up to 8 NT columns (a column is a query and a head of the KV
// head's group: all of them read the same codes) and its items, runs of tokens
// of one sequence each: every block gets an equal share of all tokens, so one
// may end in the middle of a sequence.  Each warp works alone on runs of 32 (64
// for d = 64 and where four units are held at once) tokens through its own ring of bulk copies: tokens are the M rows of both
// products, so softmax statistics stay in a lane until the end; S^T's
// accumulators become the second product's B operand by movmatrix.  The
// running maximum is raised only when a logit exceeds it by 2^8, which is
// rare, so the loop holds one vote and no reductions.  The warps' partial
// results are joined through shared memory, the blocks' of a sequence by
// attend_join_kernel in a fixed order.
//
// Measured, with the write of the new token and the join: one query of 32 heads
// over 8 x 32768 tokens (8 KV heads of 128, 285 MB) 63 us, of 28 heads over 4 x
// 131072 (4 KV heads) also 63, 58 in a graph; 44 us at the copy peak.  The loads
// alone (ring without arithmetic) take 50 us and the arithmetic alone as long:
// half of the issue slots, a third of the tensor pipe's cycles.  Start, end and
// join are 12 to 15 us of it.  Four queries of 64 heads over 8 sequences of up to
// 8192 tokens (32 columns) take 44 us, bound by the arithmetic of their columns, and
// one of 32 heads over 33 sequences of up to 8191 in groups of 32 66 us.
#include <algorithm>
#include <type_traits>

#include "kvc_kv4_attend.cuh"

namespace kvc {

int kv4_attend_read_device_error(int* out) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, tc::g_kvc_device_error, sizeof(int));
  if (e != cudaSuccess) return fail(KVC_ERR_LAUNCH, std::string("device error read: ") + cudaGetErrorString(e));
  *out = v;
  int zero = 0;
  cudaMemcpyToSymbol(tc::g_kvc_device_error, &zero, sizeof(int));
  if (v == 0) return kv4::prefill_read_device_error(out);
  return kv4::prefill_read_device_error(&zero);
}

namespace kv4 {
namespace {

constexpr float kTop = 128.0f;  // weights p s' are held as p s' hold <= 2^8 * 2^7 < 65504
constexpr uint32_t kUnheld = 127 + 100;  // exponent of 2^100: any value scale asks for less
constexpr float kLow = 2048.0f;  // a weight's second term is held so many fold, which keeps it a normal number as long as the first

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// 1 / x of a power of two within 2^-126 .. 2^126.
__device__ __forceinline__ float pow2_inverse(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }

// Powers of two, one for each of two columns and NG groups, as the bytes of their exponents.
template <int NG>
struct Pow2 {
  uint32_t word[NG == 4 ? 2 : 1];
  __device__ __forceinline__ void fill(uint32_t exponent) {
#pragma unroll
    for (uint32_t& w : word) w = exponent * 0x01010101u;
  }
  __device__ __forceinline__ float get(int j, int g) const {
    const int at = j * NG + g;
    return __uint_as_float((word[at / 4] >> (8 * (at % 4)) & 0xFFu) << 23);
  }
  __device__ __forceinline__ void set(int j, int g, float x) {
    const int at = j * NG + g, shift = 8 * (at % 4);
    word[at / 4] = (word[at / 4] & ~(0xFFu << shift)) | __float_as_uint(x) >> 23 << shift;
  }
};

// Two codes of a word as a float16 operand: nibble 0 (lo) or 1 (hi, 16 fold) of
// each half; plain codes are 2^-24 fold, centred ones c - 8.
template <bool CENTRED>
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
  if constexpr (!CENTRED) return w & 0x000F000Fu;
  uint32_t y;  // 1024 + c less 1032
  asm("sub.f16x2 %0, %1, %2;" : "=r"(y) : "r"((w & 0x000F000Fu) | 0x64006400u), "r"(0x64086408u));
  return y;
}
template <bool CENTRED>
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
  if constexpr (!CENTRED) return w & 0x00F000F0u;
  uint32_t y;  // 1024 + 16 c less 1152
  asm("sub.f16x2 %0, %1, %2;" : "=r"(y) : "r"((w & 0x00F000F0u) | 0x64006400u), "r"(0x64806480u));
  return y;
}

// The sequence of query token `tok` (the last one whose tokens start at or before it).
__device__ __forceinline__ int seq_of(const Step& S, int tok) {
  int lo = 0, hi = S.n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (S.q_start[mid] <= tok) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// NT tiles of 8 columns; TERMS float16 terms a query and a weight.
template <int D, int WPG, int NT, int TERMS>
struct Shape {
  static constexpr int NG = D / 32 / WPG;
  // Units whose logits a thread holds at once: each brings products that do not
  // wait for the others'.  Four units and 12 warps an SM beat two and 16 (one
  // query of each of 4 x 131072 tokens, 4 KV heads: 58.6 against 65.3 us).
  static constexpr int at_once = NT > 1 || NG > 2 ? 1 : D == 128 && NG == 1 && TERMS == 1 ? 4 : 2;
  static constexpr int units = at_once == 4 ? 4 : 256 / D;  // of a stage of the ring
  static constexpr int tokens = units * kUnit;
  // Registers a thread needs, roughly (accumulators, queries, columns' and
  // groups' statistics): with up to 128 an SM has 4 blocks of 4 warps, with up
  // to 168 three, else two.
  static constexpr int regs = 45 + D / 4 * NT + (NT * TERMS == 1 ? D / 8 : 0) + 10 * NT + 8 * NG * NT +
                              at_once * 4 * (NT + NG) + 35 * (TERMS - 1);
  static constexpr int warps = 4;
  static constexpr int blocks = regs < 140 ? 4 : regs < 180 ? 3 : 2;
};

template <int D, int WPG, int NT, int TERMS>
struct Smem {
  using S = Shape<D, WPG, NT, TERMS>;
  static constexpr int NG = D / 32 / WPG;
  static constexpr int stage = S::units * unit_bytes(D, NG);
  // query operands: in registers where they are few, else in shared memory
  static constexpr bool q_shared = NT * TERMS > 1;
  static constexpr int q_bytes = q_shared ? TERMS * NT * (D / 32) * 512 : 0;
  static constexpr int stages_fit = (227 * 1024 / S::blocks - 2048 - q_bytes) / (S::warps * stage);
  static constexpr int stages = stages_fit > 4 ? 4 : stages_fit;
  static constexpr int ring = S::warps * stages * stage;
  static constexpr int o_stride = D + 4;  // floats of a column: the lanes of a store meet different banks
  static constexpr int join = S::warps * 8 * NT * (o_stride + 2) * 4;
  static constexpr int q_at = ring > join ? ring : join;
  static constexpr int bytes = q_at + q_bytes;
  static_assert(stages >= 2, "stages");
};

template <int D, int WPG, int NT, int TERMS>
__global__ void __launch_bounds__(Shape<D, WPG, NT, TERMS>::warps * 32, Shape<D, WPG, NT, TERMS>::blocks)
    attend_kernel(Layout L, Step S, Split P, const uint8_t* __restrict__ pool, Qkv a, Partial part, int tile0) {
  using Sh = Shape<D, WPG, NT, TERMS>;
  using Sm = Smem<D, WPG, NT, TERMS>;
  constexpr int W = D / 32, NG = W / WPG, UB = unit_bytes(D, NG), WARPS = Sh::warps, STAGES = Sm::stages;
  constexpr int UNITS = Sh::units, TOKENS = Sh::tokens, COLS = 8 * NT, AHEAD = 32 / UNITS;
  constexpr int SUB = Sh::at_once;
  constexpr bool CENTRED = TERMS == 2;
  constexpr float kCode = CENTRED ? 1.0f : 16777216.0f;  // an operand is a code / kCode
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[WARPS][STAGES];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int h = blockIdx.y, col0 = (tile0 + (int)blockIdx.z) * COLS, group = a.n_q / L.n_kv;
  if (lane == 0)
    for (int i = 0; i < STAGES; ++i) tc::mbar_init(&full[warp][i], UNITS);
  tc::mbar_fence_init();
  __syncwarp();
  int stage = 0, parity = 0;  // the ring's next stage to read
  bool dead = false, waited = false;
  auto wait_once = [&]() {  // (what is read before is the step's own arrays and the page table)
    if (!waited) {
      grid_wait();
      grid_go();
      waited = true;
    }
  };

  for (int item = P.block_start[blockIdx.x], end = P.block_start[blockIdx.x + 1]; item < end; ++item) {
  const int4 it = P.items[item];
  const int b = it.x, t_begin = it.y, len = S.kv_len[b];
  const int q0 = S.q_start[b], n = S.q_start[b + 1] - q0, cols = n * group;
  if (col0 >= cols) continue;
  const int last = min(col0 + COLS, cols) - 1;
  const int t_end = min(it.z, visible(a.causal, len, n, last / group));
  const bool alone = P.item_start[b + 1] - P.item_start[b] == 1;
  if (t_begin > 0 && t_begin >= t_end) {  // nothing of this item is seen
    wait_once();
    for (int col = col0 + threadIdx.x; col <= last; col += WARPS * 32)
      part.ml[((int64_t)item * L.n_kv + h) * part.cols + col] = make_float2(-INFINITY, 0.0f);
    continue;
  }
  const int t_free = visible(a.causal, len, n, col0 / group);  // below it no column masks anything

  // The warp's runs of TOKENS tokens: t_begin + (warp + i WARPS) TOKENS.
  // Lane (i % AHEAD) * UNITS + u looks up unit u's page of run i and issues its
  // copy, AHEAD runs at a time, so that no copy waits for a page lookup.
  const int runs = t_end > t_begin ? (t_end - t_begin + TOKENS - 1) / TOKENS : 0;
  const int mine = runs > warp && !dead ? (runs - warp + WARPS - 1) / WARPS : 0;
  const uint32_t ring = tc::smem_u32(smem) + warp * STAGES * Sm::stage + (lane % UNITS) * UB;
  const uint8_t* src = nullptr;
  auto look = [&](int i) {  // pages of runs i .. i + AHEAD - 1
    const int run = i + lane / UNITS;  // (the position of one past the last may not fit in 32 bits)
    const int t = run < mine ? t_begin + (warp + run * WARPS) * TOKENS + (lane % UNITS) * kUnit : t_end;
    src = nullptr;
    if (t < t_end) {
      const int64_t page = page_of(L, it.w, t, &tc::g_kvc_device_error);
      // a bad entry reads page 0: its place in the sum is wrong, but in range
      src = pool + unit_off<D>(L, page < 0 ? 0 : page, h, t);
    }
  };
  auto issue = [&](int i, int stage) {
    if (i % AHEAD == 0 && i > 0) look(i);
    if (lane / UNITS == i % AHEAD) {
      uint64_t* bar = &full[warp][stage];
      if (src) {
        tc::mbar_expect_tx(bar, UB);
        tc::bulk_load(ring + stage * Sm::stage, src, UB, bar);
      } else {
        tc::mbar_arrive(bar);
      }
    }
  };
  look(0);
  wait_once();
  for (int i = 0; i < STAGES && i < mine; ++i) issue(i, (stage + i) % STAGES);

  // ---- queries: lane (r, c) holds features 32 w + 8 c + 0..7 of column r of each tile
  constexpr bool QS = Sm::q_shared;
  uint32_t qf[TERMS][QS ? 1 : NT][W][4];
  const uint32_t q_at = tc::smem_u32(smem) + Sm::q_at + lane * 16;
  float fac[NT][2], qs[NT][2][NG];
  int vis[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int col = col0 + nt * 8 + r;
    float x[W][8], top = 0.0f, sum[NG];
    const bool valid = col < cols;
    const int j = col / group;
    const int64_t at = (a.packed ? (int64_t)(q0 + j) * a.q_st : b * a.q_sb + j * a.q_st) +
                       (int64_t)(h * group + col % group) * a.q_sh + 8 * c;
#pragma unroll
    for (int g = 0; g < NG; ++g) sum[g] = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[w][e] = valid ? load_dt(a.q, at + 32 * w + e, a.dtype) : 0.0f;
        top = fmaxf(top, fabsf(x[w][e]));
        sum[w / WPG] += x[w][e];
      }
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
      for (int g = 0; g < NG; ++g) sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], o);
    }
    // 2^k with top 2^k in [2^13, 2^14): 16-bit queries are exact in float16 down
    // to 2^-28 of the row's maximum.  k is kept to +-100, where the power and
    // its inverse are normal numbers
    const int k = min(100, max(-100, 13 + 127 - (int)(__float_as_uint(top) >> 23)));
    const float up = __uint_as_float((uint32_t)(127 + k) << 23), down = __uint_as_float((uint32_t)(127 - k) << 23);
    const float sign = a.scale < 0.0f ? -up : up;  // the logits' factor is kept positive
#pragma unroll
    for (int w = 0; w < W; ++w) {
      // operand register i of word w meets the nibbles i and i + 4, of which
      // element e lies in nibble e ^ 1; nibbles 1, 3 count 16 fold
      constexpr int el[4][2] = {{1, 5}, {0, 4}, {3, 7}, {2, 6}};
      uint32_t f[TERMS][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p2 = i & 1 ? sign * 0.0625f : sign;
        const float v0 = x[w][el[i][0]] * p2, v1 = x[w][el[i][1]] * p2;
        f[0][i] = pack_half2(v0, v1);
        if constexpr (TERMS == 2) {
          const float2 hi = unpack_half2(f[0][i]);
          f[1][i] = pack_half2(v0 - hi.x, v1 - hi.y);
        }
      }
#pragma unroll
      for (int term = 0; term < TERMS; ++term)
        if constexpr (QS) {
          if (warp == nt % WARPS)
            *reinterpret_cast<uint4*>(smem + Sm::q_at + ((term * NT + nt) * W + w) * 512 + lane * 16) =
                make_uint4(f[term][0], f[term][1], f[term][2], f[term][3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) qf[term][nt][w][i] = f[term][i];
        }
    }
#pragma unroll
    for (int j2 = 0; j2 < 2; ++j2) {  // what the accumulators' columns 2 c, 2 c + 1 need
      const int from = (2 * c + j2) * 4;
      fac[nt][j2] = __shfl_sync(0xffffffffu, down, from) * kCode * fabsf(a.scale) * kLog2e;
#pragma unroll
      for (int g = 0; g < NG; ++g) qs[nt][j2][g] = __shfl_sync(0xffffffffu, sum[g] * sign, from) * (1.0f / kCode);
      const int cj = col0 + nt * 8 + 2 * c + j2;
      vis[nt][j2] = cj < cols ? visible(a.causal, len, n, cj / group) : 0;
    }
  }

  if constexpr (QS) __syncthreads();

  // Logits are kept in raw units (fac times them is log2 units).  A column's
  // reference mf (log2 units) is raised when a logit exceeds mt.
  float o[NT][2 * W][4], mf[NT][2], mt[NT][2], l[NT][2], z[NT][2][NG], zc[NT][NG][4];
  // Each column's and group's own: kTop over a power of two that the value scales
  // it has seen stay below (kUnheld: none yet).
  Pow2<NG> hold[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    hold[nt].fill(kUnheld);
#pragma unroll
    for (int i = 0; i < 2 * W; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      mf[nt][j] = mt[nt][j] = -INFINITY;
      l[nt][j] = 0.0f;
#pragma unroll
      for (int g = 0; g < NG; ++g) z[nt][j][g] = 0.0f;
    }
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) zc[nt][g][e] = 0.0f;
  }

  // SUB units at shared address `sub`, from token ts on.  MASKED: some column
  // does not see some of the tokens.
  auto absorb = [&](uint32_t sub, int ts, auto masked) {
    constexpr bool MASKED = decltype(masked)::value;
    // S^T: rows r and r + 8 of each unit, columns 2 c and 2 c + 1 of each tile
    float s[SUB][NT][4], top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      const uint32_t unit = sub + u * UB;
      uint32_t k0[W], k1[W];
      lds_words<W>(unit + k_chunk<D>(r, c), k0);
      lds_words<W>(unit + k_chunk<D>(r + 8, c), k1);
      uint32_t kp0[NG], kp1[NG];  // (scale, zero) of the rows' groups
      lds_words<NG>(unit + kp_base(D) + r * NG * 4, kp0);
      lds_words<NG>(unit + kp_base(D) + (r + 8) * NG * 4, kp1);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float acc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[nt][e] = 0.0f;
#pragma unroll
        for (int w = g * WPG; w < (g + 1) * WPG; ++w) {
          uint32_t x0 = k0[w], x1 = k1[w], qw[TERMS][NT][4];
#pragma unroll
          for (int term = 0; term < TERMS; ++term)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              if constexpr (QS) {
                lds_words<4>(q_at + ((term * NT + nt) * W + w) * 512, qw[term][nt]);
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) qw[term][nt][i] = qf[term][nt][w][i];
              }
#pragma unroll
          for (int i2 = 0; i2 < 4; i2 += 2) {
            const uint32_t a0 = codes_lo<CENTRED>(x0), a1 = codes_lo<CENTRED>(x1), a2 = codes_hi<CENTRED>(x0),
                           a3 = codes_hi<CENTRED>(x1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
              for (int term = TERMS - 1; term >= 0; --term)
                mma16816(CENTRED ? part : acc[nt], a0, a1, a2, a3, qw[term][nt][i2], qw[term][nt][i2 + 1]);
              if constexpr (CENTRED)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][e] += part[e];
            }
            x0 >>= 8;
            x1 >>= 8;
          }
        }
        const float2 p0 = unpack_half2(kp0[g]), p1 = unpack_half2(kp1[g]);
        const float off0 = CENTRED ? p0.y : fmaf(-8.0f, p0.x, p0.y), off1 = CENTRED ? p1.y : fmaf(-8.0f, p1.x, p1.y);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float off = qs[nt][e & 1][g] * (e < 2 ? off0 : off1);
            s[u][nt][e] = fmaf(acc[nt][e], e < 2 ? p0.x : p1.x, g ? s[u][nt][e] + off : off);
          }
      }
      if constexpr (MASKED) {
        const int t = ts + u * kUnit + r;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t + (e < 2 ? 0 : 8) >= vis[nt][e & 1]) s[u][nt][e] = -INFINITY;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        top[nt][0] = fmaxf(top[nt][0], fmaxf(s[u][nt][0], s[u][nt][2]));
        top[nt][1] = fmaxf(top[nt][1], fmaxf(s[u][nt][1], s[u][nt][3]));
      }
    }

    // value parameters; raise the references where they have to be
    // (all columns' value scales are the same until some are masked)
    constexpr int HN = MASKED ? NT : 1, HJ = MASKED ? 2 : 1;
    float2 vp[SUB][2][NG];
    float vtop[HN][HJ][NG];
#pragma unroll
    for (int nt = 0; nt < HN; ++nt)
#pragma unroll
      for (int j = 0; j < HJ; ++j)
#pragma unroll
        for (int g = 0; g < NG; ++g) vtop[nt][j][g] = 0.0f;
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int i2 = 0; i2 < 2; ++i2) {
        uint32_t words[NG];
        lds_words<NG>(sub + u * UB + vp_base(D, NG) + (r + 8 * i2) * NG * 4, words);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float2 p = unpack_half2(words[g]);
          vp[u][i2][g] = p;
#pragma unroll
          for (int nt = 0; nt < HN; ++nt)
#pragma unroll
            for (int j = 0; j < HJ; ++j)
              vtop[nt][j][g] = fmaxf(vtop[nt][j][g], MASKED && s[u][nt][2 * i2 + j] == -INFINITY ? 0.0f : p.x);
        }
      }
    bool raise = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) raise |= top[nt][0] > mt[nt][0] || top[nt][1] > mt[nt][1];
#pragma unroll
    for (int nt = 0; nt < HN; ++nt)
#pragma unroll
      for (int j = 0; j < HJ; ++j)
#pragma unroll
        for (int g = 0; g < NG; ++g) raise |= vtop[nt][j][g] * hold[nt].get(j, g) > kTop;
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int k = 4; k <= 16; k <<= 1) {
#pragma unroll
        for (int nt = 0; nt < HN; ++nt)
#pragma unroll
          for (int j = 0; j < HJ; ++j)
#pragma unroll
            for (int g = 0; g < NG; ++g)
              vtop[nt][j][g] = fmaxf(vtop[nt][j][g], __shfl_xor_sync(0xffffffffu, vtop[nt][j][g], k));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) top[nt][j] = fmaxf(top[nt][j], __shfl_xor_sync(0xffffffffu, top[nt][j], k));
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float f = 1.0f;
          if (top[nt][j] > mt[nt][j]) {
            const float m2 = top[nt][j] * fac[nt][j];
            f = ex2(mf[nt][j] - m2);
            mf[nt][j] = m2;
            mt[nt][j] = top[nt][j] + (fac[nt][j] > 0.0f ? kRaise / fac[nt][j] : 1.0e38f);
          }
          l[nt][j] *= f;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            z[nt][j][g] *= f;
            const float most = vtop[MASKED ? nt : 0][MASKED ? j : 0][g];
            float fg = f;
            if (const float was = hold[nt].get(j, g); most * was > kTop) {  // the next power of two above it
              const float h = kTop * 0.5f * pow2_inverse(__uint_as_float(__float_as_uint(most) & 0x7F800000u));
              fg *= h * pow2_inverse(was);
              hold[nt].set(j, g, h);
            }
#pragma unroll
            for (int i2 = 2 * g * WPG; i2 < 2 * (g + 1) * WPG; ++i2) o[nt][i2][j] *= fg, o[nt][i2][j + 2] *= fg;
            zc[nt][g][j] *= fg;
          }
        }
    }

    // weights and the second product
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      const uint32_t unit = sub + u * UB;
      uint32_t v0[W], v1[W];
      lds_words<W>(unit + v_chunk<D>(0, lane), v0);
      lds_words<W>(unit + v_chunk<D>(1, lane), v1);
      uint32_t pf[TERMS][NT][NG][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] = ex2(fmaf(s[u][nt][e], fac[nt][e & 1], -mf[nt][e & 1]));
          if (MASKED && s[u][nt][e] == -INFINITY) p[e] = 0.0f;
          l[nt][e & 1] += p[e];
        }
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int i2 = 0; i2 < 2; ++i2) {
            const float2 vs = vp[u][i2][g];
            float w0 = p[2 * i2] * (vs.x * hold[MASKED ? nt : 0].get(0, g));
            float w1 = p[2 * i2 + 1] * (vs.x * hold[MASKED ? nt : 0].get(MASKED ? 1 : 0, g));
            if constexpr (MASKED) {  // a token that a column does not see may hold NaN
              const bool n0 = s[u][nt][2 * i2] == -INFINITY, n1 = s[u][nt][2 * i2 + 1] == -INFINITY;
              w0 = n0 ? 0.0f : w0;
              w1 = n1 ? 0.0f : w1;
              z[nt][0][g] += n0 ? 0.0f : p[2 * i2] * vs.y;
              z[nt][1][g] += n1 ? 0.0f : p[2 * i2 + 1] * vs.y;
            } else {
              z[nt][0][g] = fmaf(p[2 * i2], vs.y, z[nt][0][g]);
              z[nt][1][g] = fmaf(p[2 * i2 + 1], vs.y, z[nt][1][g]);
            }
            const uint32_t hi = pack_half2(w0, w1);
            pf[0][nt][g][i2] = transpose8x8(hi);
            if constexpr (TERMS == 2) {
              const float2 got = unpack_half2(hi);
              pf[1][nt][g][i2] = transpose8x8(pack_half2((w0 - got.x) * kLow, (w1 - got.y) * kLow));
            }
          }
        if constexpr (!CENTRED) {  // the rounded weights' sums: a product with ones
#pragma unroll
          for (int g = 0; g < NG; ++g)
            mma16816(zc[nt][g], 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, pf[0][nt][g][0], pf[0][nt][g][1]);
        }
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        uint32_t y0 = v0[w], y1 = v1[w];
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
          const uint32_t a0 = codes_lo<CENTRED>(y0), a1 = codes_hi<CENTRED>(y0), a2 = codes_lo<CENTRED>(y1),
                         a3 = codes_hi<CENTRED>(y1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float part[TERMS][4] = {};
#pragma unroll
            for (int term = 0; term < TERMS; ++term)
              mma16816(CENTRED ? part[term] : o[nt][2 * w + i2], a0, a1, a2, a3, pf[term][nt][w / WPG][0],
                       pf[term][nt][w / WPG][1]);
            if constexpr (CENTRED)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][2 * w + i2][e] += fmaf(part[1][e], 1.0f / kLow, part[0][e]);
          }
          y0 >>= 8;
          y1 >>= 8;
        }
      }
    }
  };

  const uint32_t stages = tc::smem_u32(smem) + warp * STAGES * Sm::stage;
  for (int i = 0; i < mine; ++i) {
    if (__any_sync(0xffffffffu, !tc::mbar_wait(&full[warp][stage], parity, 402))) {
      // give up: wait (bounded) for the copies still in flight, then do nothing more
      for (int k = 1; k < STAGES && i + k < mine; ++k)
        tc::mbar_wait(&full[warp][(stage + k) % STAGES], parity ^ (stage + k >= STAGES), 402);
      dead = true;
      break;
    }
    const int t0 = t_begin + (warp + i * WARPS) * TOKENS;
    if (t0 + TOKENS <= t_free) {
#pragma unroll 1
      for (int u = 0; u < UNITS; u += SUB) absorb(stages + stage * Sm::stage + u * UB, t0 + u * kUnit, std::false_type{});
    } else {
#pragma unroll 1
      for (int u = 0; u < UNITS; u += SUB) absorb(stages + stage * Sm::stage + u * UB, t0 + u * kUnit, std::true_type{});
    }
    __syncwarp();  // every lane has read the stage
    if (i + STAGES < mine) {
      tc::fence_async_smem();  // the copy's writes come after those reads
      issue(i + STAGES, stage);
    }
    if (++stage == STAGES) stage = 0, parity ^= 1;
  }

  // ---- join the warps' results through shared memory
  __syncthreads();
  float* so = reinterpret_cast<float*>(smem);
  float2* sml = reinterpret_cast<float2*>(so + WARPS * COLS * Sm::o_stride);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int col = nt * 8 + 2 * c + j;
#pragma unroll
      for (int k = 4; k <= 16; k <<= 1) {
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], k);
#pragma unroll
        for (int g = 0; g < NG; ++g) z[nt][j][g] += __shfl_xor_sync(0xffffffffu, z[nt][j][g], k);
      }
      float* dst = so + (warp * COLS + col) * Sm::o_stride + 4 * r;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float unhold = pow2_inverse(hold[nt].get(j, w / WPG)), f0 = unhold * kCode, f1 = f0 * 0.0625f;
        const float zg = CENTRED ? z[nt][j][w / WPG] : fmaf(-8.0f * unhold, zc[nt][w / WPG][j], z[nt][j][w / WPG]);
        *reinterpret_cast<float4*>(dst + 32 * w) =
            make_float4(fmaf(o[nt][2 * w][j + 2], f1, zg), fmaf(o[nt][2 * w][j], f0, zg),
                        fmaf(o[nt][2 * w + 1][j + 2], f1, zg), fmaf(o[nt][2 * w + 1][j], f0, zg));
      }
      if (r == 0) sml[warp * COLS + col] = make_float2(mf[nt][j], l[nt][j]);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < COLS * (D / 4); i += WARPS * 32) {
    const int col = i / (D / 4), x = i % (D / 4) * 4, cj = col0 + col;
    if (cj >= cols) break;
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sml[w * COLS + col].x);
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float2 ml = sml[w * COLS + col];
      if (ml.y == 0.0f) continue;  // saw nothing (a sum is at least 1, or NaN)
      const float f = ex2(ml.x - top);
      const float4 v = *reinterpret_cast<const float4*>(so + (w * COLS + col) * Sm::o_stride + x);
      sum = fmaf(ml.y, f, sum);
      acc.x = fmaf(v.x, f, acc.x), acc.y = fmaf(v.y, f, acc.y), acc.z = fmaf(v.z, f, acc.z), acc.w = fmaf(v.w, f, acc.w);
    }
    if (alone) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      const int j = cj / group;
      const int64_t at = (a.packed ? (int64_t)(q0 + j) * a.o_st : b * a.o_sb + j * a.o_st) +
                         (int64_t)(h * group + cj % group) * a.o_sh + x;
      store_dt(a.out, at, acc.x * inv, a.dtype);
      store_dt(a.out, at + 1, acc.y * inv, a.dtype);
      store_dt(a.out, at + 2, acc.z * inv, a.dtype);
      store_dt(a.out, at + 3, acc.w * inv, a.dtype);
    } else {
      const int64_t at = ((int64_t)item * L.n_kv + h) * part.cols + cj;
      *reinterpret_cast<float4*>(part.o + at * D + x) = acc;
      if (x == 0) part.ml[at] = make_float2(top, sum);
    }
  }
  // the next item's copies go where the results were
  tc::fence_async_smem();
  __syncthreads();
  }
  wait_once();
}

// Joins the items of the sequences that have several.  D / 4 threads, a float4
// of features each, take a row's (a query and head's) items in turn, up to eight
// loads at once.  With few items a block of 128 threads holds G = 512 / D rows;
// with many it holds one, group g taking items g, g + G, ..., and the groups are
// added in their order.  Bound by latency: 4 to 5 us behind an attention, most
// of it the start and the trip to the partial results.
template <int D, bool WIDE>
__global__ void __launch_bounds__(128) attend_join_kernel(Layout L, Step S, Split P, Qkv a, Partial part, int64_t rows) {
  constexpr int T = D / 4, G = 128 / T, STEP = WIDE ? G : 1;
  __shared__ float4 so[G][T];
  __shared__ float ss[G];
  const int g = threadIdx.x / T, x = threadIdx.x % T;
  const int64_t id = WIDE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * G + g;
  if (id >= rows) return grid_wait();
  const int tok = (int)(id / a.n_q), head = (int)(id % a.n_q);
  const int b = seq_of(S, tok), i0 = P.item_start[b], i1 = P.item_start[b + 1];
  if (i1 - i0 <= 1) return grid_wait();
  const int j = tok - S.q_start[b], group = a.n_q / L.n_kv;
  const int h = head / group, items = i1 - i0;
  const int64_t at0 = ((int64_t)i0 * L.n_kv + h) * part.cols + j * group + head % group, step = L.n_kv * part.cols;
  grid_wait();
  float top = -INFINITY;
  for (int i = x; i < items; i += T) top = fmaxf(top, part.ml[at0 + i * step].x);
#pragma unroll
  for (int k = T / 2; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(T == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16), top, k));
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float sum = 0.0f;
  for (int i = WIDE ? g : 0; i < items; i += 8 * STEP) {
    float4 v[8];
    float2 ml[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u * STEP < items) {
        v[u] = *reinterpret_cast<const float4*>(part.o + (at0 + (i + u * STEP) * step) * D + x * 4);
        ml[u] = part.ml[at0 + (i + u * STEP) * step];
      }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u * STEP < items && ml[u].y != 0.0f) {  // 0: saw nothing
        const float f = ex2(ml[u].x - top);
        sum = fmaf(ml[u].y, f, sum);
        acc.x = fmaf(v[u].x, f, acc.x), acc.y = fmaf(v[u].y, f, acc.y);
        acc.z = fmaf(v[u].z, f, acc.z), acc.w = fmaf(v[u].w, f, acc.w);
      }
  }
  if constexpr (WIDE) {
    so[g][x] = acc;
    if (x == 0) ss[g] = sum;
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int k = 1; k < G; ++k) {
      const float4 v = so[k][x];
      acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
      sum += ss[k];
    }
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const int64_t at = (a.packed ? (int64_t)tok * a.o_st : b * a.o_sb + j * a.o_st) + (int64_t)head * a.o_sh + x * 4;
  store_dt(a.out, at, acc.x * inv, a.dtype);
  store_dt(a.out, at + 1, acc.y * inv, a.dtype);
  store_dt(a.out, at + 2, acc.z * inv, a.dtype);
  store_dt(a.out, at + 3, acc.w * inv, a.dtype);
}

template <int D>
int join(const Layout& L, const Step& S, const Split& P, const Qkv& a, const Partial& part, int64_t tokens, cudaStream_t st) {
  const int64_t rows = tokens * a.n_q;
  const bool wide = P.max_items > 8;
  const int64_t blocks = wide ? rows : ceil_div(rows, 512 / D);
  if (blocks > INT32_MAX) return fail(KVC_ERR_SHAPE, "kvc_kv4_attend: too many queries");
  return wide ? launch_after("attend_join_kernel", attend_join_kernel<D, true>, dim3((unsigned)blocks), 128, 0, st, L, S, P, a, part, rows)
              : launch_after("attend_join_kernel", attend_join_kernel<D, false>, dim3((unsigned)blocks), 128, 0, st, L, S, P, a, part, rows);
}

// 16-bit queries with more columns than this go to the kernel for many queries,
// whose time hardly depends on them up to 128 (this one's / that one's us, in a graph):
//   columns                               16          48           64           96          128
//   bfloat16
//   8 x 8192, 8 KV heads of 128      36 / 89     77 / 92     100 / 92     134 / 96     199 / 99
//   32 x 4096, the same heads       64 / 170   148 / 170    197 / 170    274 / 171    324 / 172
//   8 x 2048, 4 KV heads of 64     11.6 / 16.4 16.7 / 16.7 18.1 / 16.8  21.0 / 17.1  24.9 / 17.4
//   float16, in two terms there
//   2 x 1500, 12 KV heads of 64    10.6 / 14.7 12.9 / 14.9 14.9 / 15.1  17.0 / 15.5  18.2 / 15.8
//   8 x 8192, 8 KV heads of 128         -       77 / 141    100 / 142    134 / 145    198 / 148
//   32 x 4096, the same heads           -      147 / 266    196 / 266    273 / 267    324 / 268
constexpr int few_columns(int dtype, int head_dim) { return dtype == KVC_F16 && head_dim == 128 ? 96 : 48; }
bool many(int64_t cols, int dtype, int head_dim) { return dtype != KVC_F32 && cols > few_columns(dtype, head_dim); }

// Tiles of 8 columns a block takes.  Four, with 8 warps an SM for their
// registers, were slower than two blocks of two that read the codes twice
// (32 columns over 8 x 8192 tokens of 8 KV heads, d = 128: 66.5 against 57.4 us;
// d = 64, 4 KV heads: 27.1 against 25.8 us).
int tiles_of(int cols) { return cols <= 8 ? 1 : 2; }

template <int D, int WPG, int NT, int TERMS>
int launch(const Layout& L, const Step& S, const Split& P, const void* pool, const Qkv& a, const Partial& part,
           int64_t n_blocks, int col_tiles, cudaStream_t st) {
  using Sm = Smem<D, WPG, NT, TERMS>;
  auto kernel = attend_kernel<D, WPG, NT, TERMS>;
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_shared("attend_kernel", kernel, Sm::bytes, done)) return rc;
  for (int tile0 = 0; tile0 < col_tiles; tile0 += kGridZ) {
    const dim3 grid((unsigned)n_blocks, (unsigned)L.n_kv, (unsigned)std::min(kGridZ, col_tiles - tile0));
    if (int rc = launch_after("attend_kernel", kernel, grid, Shape<D, WPG, NT, TERMS>::warps * 32, Sm::bytes, st, L, S, P,
                              static_cast<const uint8_t*>(pool), a, part, tile0))
      return rc;
  }
  return KVC_OK;
}

template <int D, int WPG>
int launch_tiles(const Layout& L, const Step& S, const Split& P, const void* pool, const Qkv& a, const Partial& part,
                 int64_t n_blocks, int cols, cudaStream_t st) {
  const int terms = a.dtype == KVC_F32 ? 2 : 1, nt = tiles_of(cols);
  const int tiles = (int)ceil_div(cols, 8 * nt);
  if (L.n_kv > 65535) return fail(KVC_ERR_SHAPE, "kvc_kv4_attend: too many KV heads");
  if (terms == 2)
    return nt == 1 ? launch<D, WPG, 1, 2>(L, S, P, pool, a, part, n_blocks, tiles, st)
                   : launch<D, WPG, 2, 2>(L, S, P, pool, a, part, n_blocks, tiles, st);
  return nt == 1 ? launch<D, WPG, 1, 1>(L, S, P, pool, a, part, n_blocks, tiles, st)
                 : launch<D, WPG, 2, 1>(L, S, P, pool, a, part, n_blocks, tiles, st);
}

}  // namespace
}  // namespace kv4
}  // namespace kvc

using namespace kvc;
using namespace kvc::kv4;

extern "C" int kvc_kv4_attend_shape(const kvc_kv4_layout* layout, int max_new, int n_q, int dtype, int* tiles,
                                    int* resident, int* spanning) {
  if (int rc = check_layout(layout, "kvc_kv4_attend_shape")) return rc;
  if (!tiles || !resident || !spanning) return fail(KVC_ERR_ARG, "kvc_kv4_attend_shape: NULL pointer");
  if (n_q < 1 || n_q % layout->n_kv) return fail(KVC_ERR_SHAPE, "kvc_kv4_attend_shape: n_q must be a multiple of n_kv");
  const int64_t cols = std::max<int64_t>(1, (int64_t)max_new * (n_q / layout->n_kv));
  if (cols > INT32_MAX / 2) return fail(KVC_ERR_SHAPE, "kvc_kv4_attend_shape: too many queries");
  if (many(cols, dtype, layout->head_dim)) {
    *tiles = (int)prefill_tiles(cols);
    *resident = num_sms();
    *spanning = 0;
    return KVC_OK;
  }
  const int terms = dtype == KVC_F32 ? 2 : 1, nt = tiles_of((int)cols);
  *tiles = (int)ceil_div(cols, 8 * nt);
  int blocks = 0;
#define KVC_F(D, WPG)                                                                                    \
  blocks = terms == 2 ? (nt == 1 ? Shape<D, WPG, 1, 2>::blocks : Shape<D, WPG, 2, 2>::blocks)            \
                      : (nt == 1 ? Shape<D, WPG, 1, 1>::blocks : Shape<D, WPG, 2, 1>::blocks)
  KVC_KV4_DISPATCH(layout, KVC_F);
#undef KVC_F
  *resident = blocks * num_sms();
  *spanning = 1;
  return KVC_OK;
}

extern "C" size_t kvc_kv4_attend_workspace_bytes(const kvc_kv4_layout* layout, const kvc_kv4_split* split, int n_q) {
  if (!layout || !split || split->max_items <= 1 || split->n_items < 0 || split->max_new < 0 || n_q < 0) return 0;
  return (size_t)split->n_items * n_q * split->max_new * (layout->head_dim + 2) * sizeof(float);
}

extern "C" int kvc_kv4_attend(const kvc_kv4_layout* layout, const kvc_kv4_step* step, const kvc_kv4_split* split,
                              const void* pool, int n_q, const void* q, int64_t q_seq_stride, int64_t q_token_stride,
                              int64_t q_head_stride, void* out, int64_t o_seq_stride, int64_t o_token_stride,
                              int64_t o_head_stride, int packed, int dtype, int causal, float scale, void* workspace,
                              size_t ws_bytes, void* stream) {
  if (int rc = check_layout(layout, "kvc_kv4_attend")) return rc;
  if (!step || !split || !pool || !q || !out) return fail(KVC_ERR_ARG, "kvc_kv4_attend: NULL pointer");
  if (!dtype_ok(dtype)) return fail(KVC_ERR_DTYPE, "kvc_kv4_attend: bad dtype");
  if (!aligned16(pool)) return fail(KVC_ERR_ALIGN, "kvc_kv4_attend: pool not 16-byte aligned");
  if (n_q < 1 || n_q > 65535 || n_q % layout->n_kv) return fail(KVC_ERR_SHAPE, "kvc_kv4_attend: n_q must be a multiple of n_kv");
  if (step->n_tokens == 0 || split->n_items == 0) return KVC_OK;
  if (!step->rows || !step->kv_len || !step->q_start) return fail(KVC_ERR_ARG, "kvc_kv4_attend: NULL step");
  if (!split->item_start || (!many((int64_t)split->max_new * (n_q / layout->n_kv), dtype, layout->head_dim) && !split->block_start))
    return fail(KVC_ERR_ARG, "kvc_kv4_attend: NULL split");
  if (!split->items || !aligned16(split->items)) return fail(KVC_ERR_ALIGN, "kvc_kv4_attend: items not 16-byte aligned");
  if (step->n_tokens < 0 || step->n_tokens > INT32_MAX || split->max_new < 1 || split->n_items < 0 ||
      split->n_items > INT32_MAX || split->n_blocks < 0 || split->n_blocks > INT32_MAX)
    return fail(KVC_ERR_SHAPE, "kvc_kv4_attend: bad step or split sizes");
  const int64_t cols = (int64_t)split->max_new * (n_q / layout->n_kv);
  if (cols > INT32_MAX / 2) return fail(KVC_ERR_SHAPE, "kvc_kv4_attend: too many queries");
  const size_t need = kvc_kv4_attend_workspace_bytes(layout, split, n_q);
  if (need && (!workspace || ws_bytes < need || !aligned16(workspace)))
    return fail(KVC_ERR_WORKSPACE, "kvc_kv4_attend: workspace too small or not 16-byte aligned");
  const Step s{step->n_seqs, step->rows, step->kv_len, step->q_start};
  const Split p{reinterpret_cast<const int4*>(split->items), split->item_start, split->block_start, split->max_items};
  const Qkv a{q, out, q_seq_stride, q_token_stride, q_head_stride, o_seq_stride, o_token_stride, o_head_stride,
              packed, dtype, n_q, causal, scale};
  Partial part{static_cast<float*>(workspace), nullptr, cols};
  if (need) part.ml = reinterpret_cast<float2*>(part.o + (size_t)split->n_items * n_q * split->max_new * layout->head_dim);
  const Layout L = to_layout(layout);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc = KVC_OK;
  if (many(cols, dtype, layout->head_dim)) {
    rc = launch_prefill(layout, s, p, static_cast<const uint8_t*>(pool), a, part, split->n_items, st);
  } else {
#define KVC_F(D, WPG) rc = launch_tiles<D, WPG>(L, s, p, pool, a, part, split->n_blocks, (int)cols, st)
    KVC_KV4_DISPATCH(layout, KVC_F);
#undef KVC_F
  }
  if (rc || split->max_items <= 1) return rc;
  return layout->head_dim == 64 ? join<64>(L, s, p, a, part, step->n_tokens, st) : join<128>(L, s, p, a, part, step->n_tokens, st);
}
