// Attention over the pages of the 4-bit KV cache, for many queries (a prompt's
// chunk, or queries over a stored context): 16-bit queries, tcgen05.
//
// A block takes up to 256 rows of one sequence and KV head (a row is a query
// and a head of the KV head's group: they share K and V) as two tiles of 128,
// and the tokens of one item in tiles of 128 or 64.  With many rows to a token it
// pays to dequantise once into shared memory, K and V in float16 (their values are
// at most 65119), and to feed both products from there:
//   S = Q K^T    A, B in shared memory, M = N = 128, K = d
//   O += P V     A = P in TMEM (over the first half of S), B = V^T, N = d
// Roles: warps 0-3 and 4-7 hold the softmax of one row tile each (a thread a
// row: no exchanges), warps 8-11 dequantise (with 64 tokens to a tile K, and 12-15
// V), one thread of the next warp issues the products, the one after brings the
// codes by bulk copies (the last two only give up their registers: a softmax thread
// holds its row's logits).  While one tile's
// softmax runs, the tensor cores work on the other's.
//
// V lies in the cache as pairs of tokens of a feature, so V^T's rows (tokens
// contiguous) are written without a transposition; K's features lie in the
// order that its nibbles come out (1 5 0 4 3 7 2 6 of each eight), and Q's are
// put into the same order.
//
// The running maximum is a reference that is only raised when a row's logits
// exceed it by 2^8; only then O (in TMEM) is rescaled, by the softmax threads.
// Weights are held 2^7 fold in float16, so that those down to 2^-21 of the
// reference are normal numbers.  A masked token's weight is 0, but its value may be NaN:
// such values are written as 0 and their tokens flagged, and a row that does see
// a flagged token gets NaN in that group at the end.
//
// Roundings to 16 bits: weights to float16, half a step of 2^-11, and for bfloat16
// queries K and V (zero + scale q has up to 16 bits) likewise, as if the cache had
// been decoded to float16.  K's moves a logit by up to 2^-11 sum |q k|, so it grows
// with K's loud channels (as the 4 bits' own half step does, 1/30 of a group's span: 68
// times as much).  Error of the result over 1500 tokens of d = 128, where the
// output's own rounding is 1.66e-3: 1.75e-3 with channels 8 times as loud, 1.85e-3 with
// 20 times, 2.4e-3 with channels at 60, 4.2e-3 at 200; the kernel for few queries has
// none of this (its operands are the codes).  Float16 queries, whose own rounding is
// 2.0e-4, would be off by 6e-4 to 3.8e-3, so for them K and V are held in two terms:
// 2.3e-4 to 2.8e-4 on all of these.  For d = 128 the tiles then have 64 tokens, K's terms
// lie one below the other as the 128 rows of one operand, and K and V have
// dequantising warps of their own.  That costs time: 2048 queries over 8192 tokens
// 320 -> 540 us, 1001 queries of each of 2 sequences over 1500 tokens, 12 heads of 64,
// 32 -> 40 us.  Queries are held in float16 under a power of two a row.
//
// Measured: 2048 queries of 32 heads over 8192 tokens (8 KV heads of 128,
// bfloat16) 310 to 325 us as the clock allows, 740 to 780 TFLOP/s, 44 to 46% of the
// GEMM peak, and 332 with their write.  A step of 128 tokens takes about 4200 clocks,
// of which the products are 2048 (tensor pipe 46%) and the exponentials of both tiles
// 2048 (42%).  The warp that issues the products is busy or on its way through
// barriers that are open for most of the step (a wait that need not wait costs it
// about 150 clocks), with one tile's softmax 2500 from its logits' arrival to its
// last weights.  One block an SM: 227 KB of shared memory and all of TMEM.
#include <algorithm>
#include <type_traits>

#include "kvc_kv4_attend.cuh"

namespace kvc {

namespace kv4 {

int prefill_read_device_error(int* out) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, tc::g_kvc_device_error, sizeof(int));
  if (e != cudaSuccess) return fail(KVC_ERR_LAUNCH, std::string("device error read: ") + cudaGetErrorString(e));
  *out = v;
  int zero = 0;
  cudaMemcpyToSymbol(tc::g_kvc_device_error, &zero, sizeof(int));
  return KVC_OK;
}

namespace {

using namespace kvc::tc;

constexpr int kTile = 128;      // rows of a row tile
constexpr float kShift = 7.0f;  // weights are 2^7 fold

// TERMS: float16 terms of a value of K and V.  TOKENS of a token tile: 128, or 64
// where two terms of 128 features leave no room for more.
template <int D, int WPG, int TERMS>
struct Pre {
  static constexpr int W = D / 32, NG = W / WPG, UB = unit_bytes(D, NG);
  static constexpr int TOKENS = TERMS * D > 128 ? 64 : 128, UNITS = TOKENS / kUnit;
  // Two terms of 64 tokens of K lie one below the other, 128 rows of one operand: a
  // product with fewer columns takes as long (56 clocks at 64, 64 at 128).
  static constexpr bool STACKED = TOKENS == 64;
  static constexpr int K_ROWS = STACKED ? 128 : TOKENS, K_LOW = STACKED ? 64 * 128 : TOKENS * D * 2;
  static constexpr int Q = kTile * D * 2;      // bytes of a Q tile
  static constexpr int TERM = TOKENS * D * 2;  // bytes of one term of a K or V tile
  static constexpr int RAW = UNITS * UB;
  static constexpr int KV = TERMS * TERM;  // bytes of a K or V tile, its terms one after the other
  static constexpr int FLAGS = 4;  // a tile's flags outlive its codes until both softmax tiles are past it
  // Warps: 8 of the softmax, 4 that dequantise K and V in turn, or 4 for each where
  // the logits of a tile leave the registers, 4 others.  Their registers a thread
  // (40 for the others) are at most what the block was launched with.
  static constexpr bool APART = TOKENS == 64;
  static constexpr int OTHERS = APART ? 16 : 12, WARPS = OTHERS + 4;
  static constexpr int SOFTMAX_REGS = APART ? 128 : 192, DEQUANT_REGS = 88, LAUNCH_REGS = 65536 / (WARPS * 32) / 8 * 8;
  static_assert(8 * SOFTMAX_REGS + (OTHERS - 8) * DEQUANT_REGS + 4 * 40 <= WARPS * LAUNCH_REGS, "registers");
  // tiles of codes in flight; warps that dequantise both take K LEAD tiles ahead of V
  static constexpr int ROOM = 227 * 1024 - 1024 - 2 * Q - 4 * KV;
  static constexpr int RAWS = APART && 3 * RAW <= ROOM ? 3 : 2 * RAW <= ROOM ? 2 : 1, LEAD = RAWS > 1 && !APART ? 1 : 0;
  static constexpr int q = 0, k = 2 * Q, v = k + 2 * KV, raw = v + 2 * KV, flags = raw + RAWS * RAW;
  static constexpr int bars = flags + FLAGS * NG * 16;
  // barriers
  static constexpr int q_full = 0, raw_full = 2, raw_empty = raw_full + RAWS, k_full = raw_empty + RAWS,
                       v_full = k_full + 2, k_empty = v_full + 2, v_empty = k_empty + 2, s_full = v_empty + 2,
                       p_full = s_full + 2, o_done = p_full + 4, n_bars = o_done + 2;
  static constexpr int holder = bars + n_bars * 8, bytes = holder + 16;
  static_assert(bytes <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ uint32_t bits(__half2 h) {
  uint32_t r;
  memcpy(&r, &h, 4);
  return r;
}
__device__ __forceinline__ __half2 half2_of(uint32_t r) {
  __half2 h;
  memcpy(&h, &r, 4);
  return h;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t r;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// 32 columns of this thread's row, not waited for; tmem_arrived() is the wait,
// and no use of r may move before it.
__device__ __forceinline__ void tmem_fetch32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_arrived(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// z + s q, formed in float32, as two float16 terms.
__device__ __forceinline__ void two_terms(__half2 q, float2 s, float2 z, __half2& hi, __half2& lo) {
  const float2 qf = __half22float2(q);
  const float x = fmaf(qf.x, s.x, z.x), y = fmaf(qf.y, s.y, z.y);
  hi = __floats2half2_rn(x, y);
  const float2 h = __half22float2(hi);
  lo = __floats2half2_rn(x - h.x, y - h.y);
}

// Two terms where the queries can tell.
template <typename T>
constexpr int terms_of() {
  return std::is_same<T, __half>::value ? 2 : 1;
}

template <typename T, int D, int WPG>
__global__ void __launch_bounds__(Pre<D, WPG, terms_of<T>()>::WARPS * 32, 1)
    prefill_kernel(Layout L, Step S, Split P, const uint8_t* __restrict__ pool, Qkv a, Partial part, int q_vec, int o_vec,
                   int item0) {
  constexpr int TERMS = terms_of<T>();
  using C = Pre<D, WPG, TERMS>;
  constexpr int W = C::W, NG = C::NG, TOKENS = C::TOKENS;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int item = item0 + (int)blockIdx.z;
  const int4 it = P.items[item];
  const int b = it.x, t_begin = it.y, len = S.kv_len[it.x], h = blockIdx.y;
  const int q0 = S.q_start[b], n = S.q_start[b + 1] - q0, group = a.n_q / L.n_kv, rows = n * group;
  // late rows see the most tokens: they go first
  const int tiles = (rows + 2 * kTile - 1) / (2 * kTile), tile = tiles - 1 - (int)blockIdx.x;
  const int row0 = tile * 2 * kTile, last = min(row0 + 2 * kTile, rows) - 1;
  const int t_end = min(it.z, visible(a.causal, len, n, max(last, 0) / group));
  // no such rows, or nothing of this item is seen
  if (tile < 0 || (t_begin > 0 && t_begin >= t_end)) {
    grid_wait();
    grid_go();
    for (int row = row0 + threadIdx.x; tile >= 0 && row <= last; row += C::WARPS * 32)
      part.ml[((int64_t)item * L.n_kv + h) * part.cols + row] = make_float2(-INFINITY, 0.0f);
    return;
  }
  const int steps = t_end > t_begin ? (t_end - t_begin + TOKENS - 1) / TOKENS : 0;
  const int halves = row0 + kTile < rows ? 2 : 1;  // row tiles with rows

  const uint32_t base = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::bars);
  uint32_t* holder = reinterpret_cast<uint32_t*>(smem + C::holder);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::n_bars; ++i) {
      const bool per_unit = i >= C::raw_full && i < C::raw_empty;
      const bool by_mma = (i >= C::k_empty && i < C::p_full) || i >= C::o_done;
      const bool by_both = C::APART && i >= C::raw_empty && i < C::k_full;
      mbar_init(&bars[i], per_unit ? C::UNITS : by_mma ? 1 : by_both ? 2 * kTile : kTile);
    }
    mbar_fence_init();
  }
  if (warp == C::OTHERS) {
    tmem_alloc(holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *holder;
  // (what was read so far is the step's own arrays)
  grid_wait();
  grid_go();

  if (warp < 8) {
    // ---- softmax: a thread a row
    more_registers<C::SOFTMAX_REGS>();
    const int half = warp >> 2, i = threadIdx.x & (kTile - 1), row = row0 + half * kTile + i;
    if (half < halves) {
      const bool valid = row < rows;
      const int j = min(row, rows - 1) / group, g0 = min(row, rows - 1) % group;
      const int vis = visible(a.causal, len, n, j);
      const int t_free = visible(a.causal, len, n, (row0 + half * kTile) / group);  // every row of the tile sees them
      float fac;
      {  // the row of Q, a power of two and maybe a sign off, in K's order of features
        const T* src = static_cast<const T*>(a.q) + (a.packed ? (int64_t)(q0 + j) * a.q_st : b * a.q_sb + j * a.q_st) +
                       (int64_t)(h * group + g0) * a.q_sh;
        uint4 x[D / 8];
#pragma unroll
        for (int w = 0; w < D / 8; ++w) {
          x[w] = make_uint4(0, 0, 0, 0);
          if (valid && q_vec) {
            x[w] = __ldg(reinterpret_cast<const uint4*>(src) + w);
          } else if (valid) {
            T e[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = src[8 * w + k];
            memcpy(&x[w], e, 16);
          }
        }
        float top = 0.0f;
#pragma unroll
        for (int w = 0; w < D / 8; ++w) {
          T e[8];
          memcpy(e, &x[w], 16);
#pragma unroll
          for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(Elt<T>::to_f32(e[k])));
        }
        const int k2 = min(100, max(-100, 13 + 127 - (int)(__float_as_uint(top) >> 23)));
        const float up = __uint_as_float((uint32_t)(127 + k2) << 23), sign = a.scale < 0.0f ? -up : up;
        // (not 0, so that a masked logit stays -inf: a factor this small makes every weight 1)
        fac = fmaxf(__uint_as_float((uint32_t)(127 - k2) << 23) * fabsf(a.scale) * kLog2e, 1.0e-30f);
        const uint32_t qt = base + C::q + half * C::Q;
#pragma unroll
        for (int w = 0; w < D / 8; ++w) {
          T e[8];
          memcpy(e, &x[w], 16);
          float f[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = Elt<T>::to_f32(e[k]) * sign;
          sts128(qt + sw128_off(i, 8 * w, kTile), pack_half2(f[1], f[5]), pack_half2(f[0], f[4]), pack_half2(f[3], f[7]),
                 pack_half2(f[2], f[6]));
        }
        fence_async_smem();
        mbar_arrive(&bars[C::q_full + half]);
      }
      const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 TMEM lanes
      const uint32_t ts = tmem + lanes + half * kTile, to = tmem + lanes + 2 * kTile + half * D;
      float mf = -INFINITY, mt = -INFINITY;
      uint64_t l2 = f2_pack(0.0f, 0.0f);
      uint32_t poison = 0;
      bool ok = true;

      for (int step = 0; step < steps; ++step) {
        // (the flags of these tokens were written before K's barrier, which the
        // issuing thread waited for before it issued S)
        ok = ok && mbar_wait(&bars[C::s_full + half], step & 1, 411);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        const int seen = vis - (t_begin + step * TOKENS);  // columns below it are seen
        uint32_t r[TOKENS / 32][32];
#pragma unroll
        for (int ch = 0; ch < TOKENS / 32; ++ch) tmem_fetch32(ts + ch * 32, r[ch]);
#pragma unroll
        for (int ch = 0; ch < TOKENS / 32; ++ch) tmem_arrived(r[ch]);
        if constexpr (C::STACKED) {
#pragma unroll
          for (int ch = 0; ch < TOKENS / 32; ++ch) {
            uint32_t low[32];
            tmem_fetch32(ts + TOKENS + ch * 32, low);
            tmem_arrived(low);
#pragma unroll
            for (int k = 0; k < 32; ++k) r[ch][k] = __float_as_uint(__uint_as_float(r[ch][k]) + __uint_as_float(low[k]));
          }
        }
        if (t_begin + (step + 1) * TOKENS > t_free) {
#pragma unroll
          for (int ch = 0; ch < TOKENS / 32; ++ch)
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (ch * 32 + k >= seen) r[ch][k] = 0xFF800000u;  // -inf
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < TOKENS / 4; k += 2)
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) {
            const int at = ch * (TOKENS / 4) + k;
            tops[ch] = fmaxf(tops[ch], fmaxf(__uint_as_float(r[at / 32][at % 32]), __uint_as_float(r[at / 32][at % 32 + 1])));
          }
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const bool raise = top > mt;
        if (__any_sync(0xffffffffu, raise)) {
          float f = 1.0f;
          if (raise) {
            const float m2 = top * fac - kShift;
            f = ex2(mf - m2);
            mf = m2;
            mt = top + kRaise / fac;
          }
          l2 = f2_mul(l2, f2_pack(f, f));
          if (step > 0) {
            ok = ok && mbar_wait(&bars[C::o_done + half], (step - 1) & 1, 410);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
#pragma unroll 1
            for (int ch = 0; ch < D / 16; ++ch) {
              uint32_t o[16];
              tmem_ld16(to + ch * 16, o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tmem_st16(to + ch * 16, o);
            }
          }
        }
        const float off = mf == -INFINITY ? 0.0f : -mf;  // (nothing seen yet: every logit is -inf)
        const uint64_t fac2 = f2_pack(fac, fac), off2 = f2_pack(off, off);
#pragma unroll
        for (int hf = 0; hf < TOKENS / 64; ++hf) {
          uint32_t p[32];
#pragma unroll
          for (int k = 0; k < 64; k += 2) {
            const uint32_t* at = &r[2 * hf + k / 32][k % 32];
            float x, y;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(at[0]), __uint_as_float(at[1])), fac2, off2), x, y);
            x = ex2(x);
            y = ex2(y);
            l2 = f2_add(l2, f2_pack(x, y));
            p[k / 2] = pack_half2(x, y);
          }
          tmem_st32(ts + hf * 32, p);
          // the product with the first 64 tokens starts while the others' weights are formed
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&bars[C::p_full + 2 * half + hf]);
        }
        // values that are NaN were written as 0: remember the rows that see them
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          uint32_t fl[TOKENS / 32], any = 0;
          lds_words<TOKENS / 32>(base + C::flags + ((step % C::FLAGS) * NG + g) * 16, fl);
#pragma unroll
          for (int k = 0; k < TOKENS / 32; ++k) any |= fl[k];
          if (any) {
#pragma unroll
            for (int k = 0; k < TOKENS / 32; ++k) {
              const int m = seen - 32 * k;
              if (m > 0 && (fl[k] & (m >= 32 ? 0xFFFFFFFFu : (1u << m) - 1u))) poison |= 1u << g;
            }
          }
        }
      }

      // ---- the row's result
      float l, l1;
      f2_unpack(l2, l, l1);
      l += l1;
      if (steps > 0) ok = ok && mbar_wait(&bars[C::o_done + half], (steps - 1) & 1, 413);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      const bool alone = P.item_start[b + 1] - P.item_start[b] == 1;
      const float inv = l == 0.0f ? 0.0f : alone ? 1.0f / l : 1.0f;
      const int64_t at = alone ? (a.packed ? (int64_t)(q0 + j) * a.o_st : b * a.o_sb + j * a.o_st) + (int64_t)(h * group + g0) * a.o_sh
                               : (((int64_t)item * L.n_kv + h) * part.cols + row) * D;
#pragma unroll
      for (int ch = 0; ch < D / 32; ++ch) {
        float o[32];
        __syncwarp();
        if (steps > 0) tmem_ld32(to + ch * 32, o);
        const bool bad = (poison >> (ch / WPG)) & 1;
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = bad ? __uint_as_float(0x7FC00000u) : l == 0.0f ? 0.0f : o[k] * inv;
        if (valid && alone && o_vec) {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at + ch * 32);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            T e[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) e[x] = Elt<T>::from(o[8 * k + x]);
            uint4 y;
            memcpy(&y, e, 16);
            dst[k] = y;
          }
        } else if (valid && alone) {
#pragma unroll
          for (int k = 0; k < 32; ++k) static_cast<T*>(a.out)[at + ch * 32 + k] = Elt<T>::from(o[k]);
        } else if (valid) {
          float4* dst = reinterpret_cast<float4*>(part.o + at + ch * 32);
#pragma unroll
          for (int k = 0; k < 8; ++k) dst[k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
        }
      }
      if (valid && !alone) part.ml[at / D] = make_float2(mf, l);
      tc_fence_before();
    }
  } else if (warp < C::OTHERS) {
    // ---- dequantise: 128 threads, or 128 for K and 128 for V
    fewer_registers<C::DEQUANT_REGS>();
    const int w4 = warp & 3;
    bool ok = true;
    // K: a thread takes chunk c of four tokens, 32 apart.  Eight lanes of a store
    // hold tokens t and t + 4, whose swizzles differ: no two meet a bank.
    const int c = lane & 3, t = w4 * 8 + ((lane >> 2) & 1) * 4 + (lane >> 3);
    const uint32_t k_src = base + C::raw + (t >> 4) * C::UB + k_chunk<D>(t & 15, c);
    const uint32_t kp_src = base + C::raw + (t >> 4) * C::UB + kp_base(D) + (t & 15) * NG * 4;
    uint32_t k_dst[2];  // of words w with w % 2 = 0, 1
#pragma unroll
    for (int w = 0; w < 2; ++w) k_dst[w] = base + C::k + sw128_off(t, 32 * w + 8 * c, C::K_ROWS);
    // V^T: a thread takes eight tokens (16-byte chunk q8 of a row) of the features
    // 32 u + 4 r + 0..3 of VW words u, from u0 on (all of them, or half where a tile has
    // 8 chunks and not 16)
    constexpr int VW = W * TOKENS / 128;
    const int q8 = ((lane & 3) | ((lane >> 3) << 2)) & (TOKENS / 8 - 1), r = ((lane >> 2) & 1) | (w4 << 1);
    const int u0 = VW < W ? (lane >> 4) * VW : 0;
    const uint32_t v_src = base + C::raw + (q8 >> 1) * C::UB + v_chunk<D>(q8 & 1, r * 4) + u0 * 4;
    const uint32_t vp_src = base + C::raw + (q8 >> 1) * C::UB + vp_base(D, NG) + (q8 & 1) * 8 * NG * 4;
    uint32_t v_dst[4];  // of the features with f % 4 = 0..3
#pragma unroll
    for (int k = 0; k < 4; ++k) v_dst[k] = base + C::v + sw128_off(4 * r + k, 8 * q8, D) + u0 * 4096;

    // The step's K, and the flags of the tokens whose values are NaN; whether V has to
    // look for such tokens or for ones past the end.
    auto take_k = [&](int step) -> bool {
      const int buf = step & 1, t0 = t_begin + step * TOKENS;
      const uint32_t raw = step % C::RAWS * C::RAW, tile_at = buf * C::KV;
      bool dirty = t0 + TOKENS > t_end;
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int k = 0; k < TOKENS / 32; ++k) {
          const int tok = 32 * k + lane;
          const uint32_t p = lds32(base + C::raw + raw + (tok >> 4) * C::UB + vp_base(D, NG) + ((tok & 15) * NG + g) * 4);
          const bool nan = __hisnan(__low2half(half2_of(p))) || __hisnan(__high2half(half2_of(p)));
          const uint32_t fl = __ballot_sync(0xffffffffu, nan && t0 + tok < t_end);
          dirty |= fl != 0;
          if (threadIdx.x == 8 * 32)
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(base + C::flags + ((step % C::FLAGS) * NG + g) * 16 + k * 4), "r"(fl)
                         : "memory");
        }
#pragma unroll 1  // (unrolled, its loads spill: 2048 queries over 8192 tokens 314 -> 320 us)
      for (int rep = 0; rep < TOKENS / 32; ++rep) {
        uint32_t x[W];
        lds_words<W>(k_src + raw + rep * 2 * C::UB, x);
        __half2 s2, z2;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          if (w % WPG == 0) {
            const __half2 sz = half2_of(lds32(kp_src + raw + rep * 2 * C::UB + w / WPG * 4));
            s2 = __low2half2(sz), z2 = __high2half2(sz);
          }
          const uint32_t y = x[w] >> 8, at = k_dst[w & 1] + tile_at + (w >> 1) * (C::K_ROWS * 128) + rep * 4096;
          const __half2 q[4] = {centred_lo(x[w]), centred_hi(x[w]), centred_lo(y), centred_hi(y)};
          __half2 hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (TERMS == 2) two_terms(q[e], __half22float2(s2), __half22float2(z2), hi[e], lo[e]);
            else hi[e] = __hfma2(q[e], s2, z2);
          }
          sts128(at, bits(hi[0]), bits(hi[1]), bits(hi[2]), bits(hi[3]));
          if constexpr (TERMS == 2) sts128(at + C::K_LOW, bits(lo[0]), bits(lo[1]), bits(lo[2]), bits(lo[3]));
        }
      }
      if constexpr (C::APART) mbar_arrive(&bars[C::raw_empty + step % C::RAWS]);
      fence_async_smem();
      mbar_arrive(&bars[C::k_full + buf]);
      return dirty;
    };
    auto take_v = [&](int step, bool check) {
      const int buf = step & 1, t0 = t_begin + step * TOKENS;
      const uint32_t raw = step % C::RAWS * C::RAW, tile_at = buf * C::KV;
      uint32_t x[4][VW];
#pragma unroll
      for (int k = 0; k < 4; ++k) lds_words<VW>(v_src + raw + k * (v_chunk<D>(0, 1) - v_chunk<D>(0, 0)), x[k]);
      __half2 s2[4], z2[4];
#pragma unroll
      for (int u = 0; u < VW; ++u) {
        if (u % WPG == 0) {
          uint32_t p[8];
          if constexpr (NG == 1) {
            uint32_t p0[4], p1[4];
            lds_words<4>(vp_src + raw, p0);
            lds_words<4>(vp_src + raw + 16, p1);
#pragma unroll
            for (int k = 0; k < 4; ++k) p[k] = p0[k], p[4 + k] = p1[k];
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) p[k] = lds32(vp_src + raw + (k * NG + (u0 + u) / WPG) * 4);
          }
          if (check) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const __half2 h = half2_of(p[k]);
              if (__hisnan(__low2half(h)) || __hisnan(__high2half(h)) || t0 + 8 * q8 + k >= t_end) p[k] = 0;
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            s2[k] = __lows2half2(half2_of(p[2 * k]), half2_of(p[2 * k + 1]));
            z2[k] = __highs2half2(half2_of(p[2 * k]), half2_of(p[2 * k + 1]));
          }
        }
        // nibbles 0..3 are features 1, 0, 3, 2
        uint32_t o[TERMS][4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t y = x[k][u] >> 8;
          const __half2 q[4] = {centred_hi(x[k][u]), centred_lo(x[k][u]), centred_hi(y), centred_lo(y)};
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            if constexpr (TERMS == 2) {
              __half2 hi, lo;
              two_terms(q[f], __half22float2(s2[k]), __half22float2(z2[k]), hi, lo);
              o[0][f][k] = bits(hi), o[1][f][k] = bits(lo);
            } else {
              o[0][f][k] = bits(__hfma2(q[f], s2[k], z2[k]));
            }
          }
        }
#pragma unroll
        for (int term = 0; term < TERMS; ++term)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            sts128(v_dst[k] + tile_at + term * C::TERM + u * 4096, o[term][k][0], o[term][k][1], o[term][k][2], o[term][k][3]);
      }
      mbar_arrive(&bars[C::raw_empty + step % C::RAWS]);
      fence_async_smem();
      mbar_arrive(&bars[C::v_full + buf]);
    };
    auto wait_raw = [&](int step) { return mbar_wait(&bars[C::raw_full + step % C::RAWS], (step / C::RAWS) & 1, 420); };
    auto wait_k = [&](int step) { return step < 2 || mbar_wait(&bars[C::k_empty + (step & 1)], ((step >> 1) + 1) & 1, 421); };
    auto wait_v = [&](int step) { return step < 2 || mbar_wait(&bars[C::v_empty + (step & 1)], ((step >> 1) + 1) & 1, 422); };
    if constexpr (C::APART) {
      const bool for_k = warp < 12;
      for (int step = 0; step < steps; ++step) {
        ok = wait_raw(step) && (for_k ? wait_k(step) : wait_v(step));
        if (!__all_sync(0xffffffffu, ok)) break;
        if (for_k) take_k(step);
        else take_v(step, true);
      }
    } else {
      // K goes one tile ahead of V where two tiles of codes fit: the scores of the next
      // tile are issued before the product with this one's V.
      bool dirty = false;
      for (int it = 0; it < steps + C::LEAD; ++it) {
        const bool check = dirty;
        if (it < steps) {
          ok = wait_raw(it) && wait_k(it);
          if (!__all_sync(0xffffffffu, ok)) break;
          dirty = take_k(it);
        }
        if (it >= C::LEAD) {
          ok = wait_v(it - C::LEAD);
          if (!__all_sync(0xffffffffu, ok)) break;
          take_v(it - C::LEAD, C::LEAD ? check : dirty);
        }
      }
    }
  } else {
    fewer_registers<40>();
    if (warp == C::OTHERS) {
      // ---- issue the products.  The whole warp walks the loop with uniform values
      // and one elected lane issues: a product takes 64 cycles, so there is time
      // for few instructions between two of them
      constexpr uint32_t id_s = idesc_f16(kTile, C::K_ROWS, false), id_o = idesc_f16(kTile, D, false);
      const uint64_t q_desc = desc_sw128(base + C::q), k_desc = desc_sw128(base + C::k), v_desc = desc_sw128(base + C::v);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      bool ok = true;
      auto scores = [&](int half, int step) {
        const uint64_t qd = q_desc + (uint32_t)half * (C::Q >> 4), kd = k_desc + (uint32_t)(step & 1) * (C::KV >> 4);
        if (elect_one()) {
#pragma unroll
          for (int term = 0; term < (C::STACKED ? 1 : TERMS); ++term)
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const uint32_t q_off = ((ks >> 2) * (kTile * 128) + (ks & 3) * 32) >> 4;
              const uint32_t k_off = (term * C::K_LOW + (ks >> 2) * (C::K_ROWS * 128) + (ks & 3) * 32) >> 4;
              umma_f16(tm + half * kTile, qd + q_off, kd + k_off, id_s, ks || term ? 1u : 0u);
            }
          umma_commit(&bars[C::s_full + half]);
        }
        __syncwarp();
      };
      if (steps > 0) {
        for (int half = 0; half < halves; ++half) ok = ok && mbar_wait(&bars[C::q_full + half], 0, 430);
        ok = ok && mbar_wait(&bars[C::k_full], 0, 431);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        if (ok) {
          for (int half = 0; half < halves; ++half) scores(half, 0);
          if (steps > 2 && elect_one()) umma_commit(&bars[C::k_empty]);
          __syncwarp();
        }
      }
      for (int step = 0; ok && step < steps; ++step) {
        ok = mbar_wait(&bars[C::v_full + (step & 1)], (step >> 1) & 1, 432);
        const uint64_t vd = v_desc + (uint32_t)(step & 1) * (C::KV >> 4);
        for (int half = 0; half < halves; ++half) {
#pragma unroll
          for (int hf = 0; hf < TOKENS / 64; ++hf) {
            ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars[C::p_full + 2 * half + hf], step & 1, 434));
            tc_fence_after();
            if (ok && elect_one()) {
#pragma unroll
              for (int term = 0; term < TERMS; ++term)
#pragma unroll
                for (int ks = 0; ks < 64 / 16; ++ks)
                  umma_f16_ts(tm + 2 * kTile + half * D, tm + half * kTile + hf * 32 + ks * 8,
                              vd + ((term * C::TERM + hf * (D * 128) + ks * 32) >> 4), id_o,
                              step || hf || ks || term ? 1u : 0u);
              if (hf == TOKENS / 64 - 1) umma_commit(&bars[C::o_done + half]);
            }
            __syncwarp();
          }
          if (half == 0 && step + 1 < steps) {
            ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars[C::k_full + ((step + 1) & 1)], ((step + 1) >> 1) & 1, 433));
            tc_fence_after();
          }
          if (ok && step + 1 < steps) scores(half, step + 1);
        }
        // only where somebody waits: none may be on its way when the block ends
        if (ok && elect_one()) {
          if (step + 2 < steps) umma_commit(&bars[C::v_empty + (step & 1)]);
          if (step + 3 < steps) umma_commit(&bars[C::k_empty + ((step + 1) & 1)]);
        }
        __syncwarp();
      }
    } else if (warp == C::OTHERS + 1) {
      // ---- bring the codes: lane u copies unit u of each tile
      bool ok = true;
      auto page = [&](int step) -> const uint8_t* {
        if (lane >= C::UNITS || step >= steps) return nullptr;  // (the position may not fit in 32 bits)
        const int t = t_begin + step * TOKENS + lane * kUnit;
        if (t >= t_end) return nullptr;
        const int64_t p = page_of(L, it.w, t, &g_kvc_device_error);
        return pool + unit_off<D>(L, p < 0 ? 0 : p, h, t);  // a bad entry reads page 0: wrong, but in range
      };
      const uint8_t* src = page(0);
      for (int step = 0; step < steps; ++step) {
        const uint8_t* next = page(step + 1);
        const int rs = step % C::RAWS;
        if (step >= C::RAWS) ok = mbar_wait(&bars[C::raw_empty + rs], (step / C::RAWS + 1) & 1, 440);
        if (!__all_sync(0xffffffffu, ok)) break;
        fence_async_smem();  // the copies' writes come after the reads that freed the place
        if (lane < C::UNITS) {
          if (src) {
            mbar_expect_tx(&bars[C::raw_full + rs], C::UB);
            bulk_load(base + C::raw + rs * C::RAW + lane * C::UB, src, C::UB, &bars[C::raw_full + rs]);
          } else {
            mbar_arrive(&bars[C::raw_full + rs]);
          }
        }
        src = next;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == C::OTHERS) tmem_dealloc(tmem, 512);
}

template <typename T, int D, int WPG>
int launch(const Layout& L, const Step& S, const Split& P, const uint8_t* pool, const Qkv& a, const Partial& part,
           int64_t tiles, int64_t n_items, cudaStream_t st) {
  using C = Pre<D, WPG, terms_of<T>()>;
  auto kernel = prefill_kernel<T, D, WPG>;
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_shared("prefill_kernel", kernel, C::bytes, done)) return rc;
  // the warps' shares of the registers add up to the launch's: with fewer they would wait for good
  static const int regs = [&] {
    cudaFuncAttributes at{};
    return cudaFuncGetAttributes(&at, kernel) == cudaSuccess ? at.numRegs : 0;
  }();
  if (regs != C::LAUNCH_REGS) return fail(KVC_ERR_UNSUPPORTED, "prefill_kernel: not built with its registers");
  const int q_vec = aligned16(a.q) && ((a.q_sb | a.q_st | a.q_sh) & 7) == 0;
  const int o_vec = aligned16(a.out) && ((a.o_sb | a.o_st | a.o_sh) & 7) == 0;
  for (int64_t item0 = 0; item0 < n_items; item0 += kGridZ) {
    const dim3 grid((unsigned)tiles, (unsigned)L.n_kv, (unsigned)std::min<int64_t>(kGridZ, n_items - item0));
    if (int rc = launch_after("prefill_kernel", kernel, grid, C::WARPS * 32, C::bytes, st, L, S, P, pool, a, part, q_vec, o_vec,
                              (int)item0))
      return rc;
  }
  return KVC_OK;
}

}  // namespace

int launch_prefill(const kvc_kv4_layout* l, const Step& S, const Split& P, const uint8_t* pool, const Qkv& a,
                   const Partial& part, int64_t n_items, cudaStream_t st) {
  const Layout L = to_layout(l);
  const int64_t tiles = prefill_tiles(part.cols);
  if (L.n_kv > 65535) return fail(KVC_ERR_SHAPE, "kvc_kv4_attend: too many KV heads");
  int rc = KVC_OK;
#define KVC_F(D, WPG)                                                                             \
  rc = a.dtype == KVC_F16 ? launch<__half, D, WPG>(L, S, P, pool, a, part, tiles, n_items, st)              \
                          : launch<__nv_bfloat16, D, WPG>(L, S, P, pool, a, part, tiles, n_items, st)
  KVC_KV4_DISPATCH(l, KVC_F);
#undef KVC_F
  return rc;
}

}  // namespace kv4
}  // namespace kvc
