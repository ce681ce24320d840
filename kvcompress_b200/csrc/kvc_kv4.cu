// Writing, reading and moving the pages of the 4-bit KV cache.
//
// Figures are for one layer of 32768 tokens, 8 heads of 128, bf16, one group a
// head: 134 MB dense and 36 MB packed, 26 us at the copy peak of 6.55 TB/s.  The
// write takes 47.5 us (3.6 TB/s): it forms 67M exactly rounded codes at 16
// instructions each, which fill 65% of the issue slots over the whole launch; the
// rest are waits for its inputs.  The read takes 27 us (6.3 TB/s), bound by memory;
// page copies reach 96% of the copy peak.  A warp of the write and read kernels takes 8
// tokens of one head's K and V, 4 lanes a token: lane c of a token holds the
// features 32 w + 8 c + 0..7, which is both a 16-byte load of a 16-bit input
// (4 lanes: 64 contiguous bytes) and word w of K's chunk c, so K's codes need
// no exchange at all and V's one shuffle a word with the neighbouring token.
#include <algorithm>
#include <type_traits>

#include "kvc_kv4.cuh"
#include "kvc_tc.cuh"

namespace kvc {

int kv4_read_device_error(int* out) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, tc::g_kvc_device_error, sizeof(int));
  if (e != cudaSuccess) return fail(KVC_ERR_LAUNCH, std::string("device error read: ") + cudaGetErrorString(e));
  *out = v;
  int zero = 0;
  cudaMemcpyToSymbol(tc::g_kvc_device_error, &zero, sizeof(int));
  return KVC_OK;
}

namespace kv4 {
namespace {

// ---- element access ---------------------------------------------------------

// Eight consecutive elements: as they lie in memory (packed pairs of 16-bit
// ones, so that a warp holds K and V at once), and as float32.
template <typename T>
struct Eight {
  static constexpr int N = sizeof(T) * 2;  // 32-bit words
  uint32_t r[N];

  __device__ __forceinline__ void load(const T* p, bool vec) {  // vec: 16-byte aligned
    if (vec) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p) + i / 4);
        r[i] = a.x, r[i + 1] = a.y, r[i + 2] = a.z, r[i + 3] = a.w;
      }
    } else {
      T e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
      memcpy(r, e, sizeof r);
    }
  }
  __device__ __forceinline__ void floats(float (&x)[8]) const {
    T e[8];
    memcpy(e, r, sizeof r);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elt<T>::to_f32(e[i]);
  }
};

// Smallest and largest of several Eights (NaN left out), and 0 if all are
// finite, else NaN; 16-bit elements two at a time.
template <typename T, int W>
__device__ __forceinline__ void extremes(const Eight<T>* x, float& lo, float& hi, float& odd) {
  if constexpr (sizeof(T) == 4) {
    lo = hi = __uint_as_float(x[0].r[0]);
    odd = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float a = __uint_as_float(x[w].r[i]), b = __uint_as_float(x[w].r[i + 1]);
        lo = fminf(lo, fminf(a, b));
        hi = fmaxf(hi, fmaxf(a, b));
        odd = fmaf(b, 0.0f, fmaf(a, 0.0f, odd));
      }
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 l, h, o, zero;
    memcpy(&l, &x[0].r[0], 4);
    h = l;
    const uint32_t none = 0;
    memcpy(&zero, &none, 4);
    o = zero;
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        T2 v;
        memcpy(&v, &x[w].r[i], 4);
        l = __hmin2(l, v);
        h = __hmax2(h, v);
        o = __hfma2(v, zero, o);
      }
    T a[2];
    memcpy(a, &l, 4);
    lo = fminf(Elt<T>::to_f32(a[0]), Elt<T>::to_f32(a[1]));
    memcpy(a, &h, 4);
    hi = fmaxf(Elt<T>::to_f32(a[0]), Elt<T>::to_f32(a[1]));
    memcpy(a, &o, 4);
    odd = Elt<T>::to_f32(a[0]) + Elt<T>::to_f32(a[1]);
  }
}

// (Streaming stores: dense K and V are larger than what is worth keeping in L2;
// one layer of 32768 tokens: 30.9 -> 26.8 us.)
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
    __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(x[4], x[5], x[6], x[7]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T e[2] = {Elt<T>::from(x[2 * i]), Elt<T>::from(x[2 * i + 1])};
      memcpy(&w[i], e, 4);
    }
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// ---- the quantiser ------------------------------------------------------------

// scale = (hi - lo) / 15 and zero = lo + 8 scale, each rounded to float32 and then
// to float16.  One float32 operation rounds its exact result once: the sum
// always, the quotient where hi - lo is exact, as it nearly always is for 16-bit
// elements; elsewhere the quotient is formed in 64 bits.  A NaN in the group
// makes both NaN.
__device__ __forceinline__ __half2 params_of(float lo, float hi, bool nan) {
  if (nan) return __half2half2(__ushort_as_half(0x7FFF));
  const float d = hi - lo, bb = d - hi, err = (hi - (d - bb)) + (-lo - bb);  // two-sum: d + err = hi - lo
  float q = __fdiv_rn(d, 15.0f);
  if (err != 0.0f) q = (float)(((double)hi - (double)lo) / 15.0);
  const __half s = __float2half_rn(q);
  const __half z = __float2half_rn(__fadd_rn(lo, 8.0f * __half2float(s)));
  return __halves2half2(s, z);
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Codes 0..15: clamp(rint((x - z) / s), -8, 7) + 8 of the exact quotient.
//
// In float32, v = sat((x - z) / (15 s) + 8 / 15) is the code over 15, and 15 v +
// 1.5 2^23 rounds it to an integer; the distance from there, 15 v - n, says how
// near a half it was.  The roundings make an error below 4e-6, so only a
// distance above 0.49999 needs more: there the sign of (x - z) - (n + 1/2) s
// decides, which is exact: (n + 1/2) s has 16 bits, the rounded x - z is next to
// it (their difference is exact by Sterbenz' lemma), and the rounding error of
// x - z is itself a float32 (Knuth's two-sum).  A NaN gives 0.
constexpr float kMagic = 12582912.0f;

__device__ __noinline__ float code_near_half(float x, float s, float z, float t) {
  const float f = floorf(t) - 8.0f, h = (f + 0.5f) * s;
  const float a = x - z, bb = a - x;
  const float err = (x - (a - bb)) + (-z - bb);
  const float res = (a - h) + err;
  const bool odd = (((int)f) & 1) != 0;
  return (res > 0.0f || (res == 0.0f && odd) ? f + 1.0f : f) + 8.0f;
}

// The word of eight elements (the first of each byte in its high nibble).
__device__ __forceinline__ uint32_t word_of(const float (&x)[8], float s, float z, float inv15) {
  using namespace tc;
  const uint64_t z2 = f2_pack(-z, -z), c15 = f2_pack(15.0f, 15.0f), m15 = f2_pack(-15.0f, -15.0f),
                 magic = f2_pack(kMagic, kMagic), unmagic = f2_pack(-kMagic, -kMagic);
  float n[8], t[8], far = 0.0f;  // n: the codes, negative
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    float a, b;
    f2_unpack(f2_add(f2_pack(x[e], x[e + 1]), z2), a, b);
    t[e] = __saturatef(fmaf(a, inv15, 8.0f / 15.0f));
    t[e + 1] = __saturatef(fmaf(b, inv15, 8.0f / 15.0f));
    const uint64_t t2 = f2_pack(t[e], t[e + 1]), n2 = f2_add(f2_fma(t2, m15, magic), unmagic);
    f2_unpack(n2, n[e], n[e + 1]);
    f2_unpack(f2_fma(t2, c15, n2), a, b);
    far = fmaxf(far, fmaxf(fabsf(a), fabsf(b)));
  }
  if (far > 0.49999f) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (fabsf(fmaf(t[e], 15.0f, n[e])) > 0.49999f) n[e] = -code_near_half(x[e], s, z, t[e] * 15.0f);
  }
  // four codes are an integer below 2^16, exact in float32
  const float lo = kMagic - fmaf(fmaf(fmaf(n[2], 16.0f, n[3]), 16.0f, n[0]), 16.0f, n[1]);
  const float hi = kMagic - fmaf(fmaf(fmaf(n[6], 16.0f, n[7]), 16.0f, n[4]), 16.0f, n[5]);
  return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x5410);
}

struct KvIn {
  const void *k, *v;
  int64_t sb, st, sh;  // strides of a sequence, a token and a head, in elements
  int packed;          // tokens of all sequences in one row of tokens (sb unused)
  int vec;             // 16-byte loads are aligned
};

// Quantise this lane's W words: their codes, and the parameters of its token's
// groups.
template <typename T, int W, int WPG>
__device__ __forceinline__ void quantise(const Eight<T> (&x)[W], uint32_t (&word)[W], __half2 (&par)[W / WPG]) {
#pragma unroll
  for (int g = 0; g < W / WPG; ++g) {
    float lo, hi, odd;
    extremes<T, WPG>(&x[g * WPG], lo, hi, odd);
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const bool rare = __any_sync(0xffffffffu, !(odd == 0.0f) || lo < -kLimit || hi > kLimit);
    bool nan = false;
    if (rare) {
#pragma unroll
      for (int w = 0; w < WPG; ++w) {
        float f[8];
        x[g * WPG + w].floats(f);
#pragma unroll
        for (int e = 0; e < 8; ++e) nan |= f[e] != f[e];
      }
      nan |= __shfl_xor_sync(0xffffffffu, (int)nan, 1) != 0;
      nan |= __shfl_xor_sync(0xffffffffu, (int)nan, 2) != 0;
      lo = fminf(fmaxf(lo, -kLimit), kLimit);
      hi = fminf(fmaxf(hi, -kLimit), kLimit);
    }
    par[g] = params_of(lo, hi, nan);
    const float s = __low2float(par[g]), z = __high2float(par[g]), inv15 = s > 0.0f ? rcp_approx(15.0f * s) : 0.0f;
#pragma unroll
    for (int w = g * WPG; w < (g + 1) * WPG; ++w) {
      float f[8];
      x[w].floats(f);
      if (rare) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = fminf(fmaxf(f[e], -kLimit), kLimit);
      }
      word[w] = word_of(f, s, z, inv15);
    }
  }
}

template <int W>
__device__ __forceinline__ void store_words(uint8_t* dst, const uint32_t (&word)[W]) {
  if constexpr (W == 4) *reinterpret_cast<uint4*>(dst) = make_uint4(word[0], word[1], word[2], word[3]);
  else *reinterpret_cast<uint2*>(dst) = make_uint2(word[0], word[1]);
}

// W = D / 32 words a lane; WPG words a quantisation group.  K and V of a token
// share a warp: twice the loads in flight (a warp each: 62 us instead of 50).  Seven
// blocks an SM where a lane's inputs are 16-bit (72 registers): 50 -> 47.5 us.
template <typename T, int D, int WPG>
__global__ void __launch_bounds__(128, sizeof(T) == 2 ? 7 : 1) kv4_write_kernel(Layout L, Step S, uint8_t* pool, KvIn in, int n_halves,
                                                        const int32_t* __restrict__ half_seq,
                                                        const int32_t* __restrict__ half_start) {
  constexpr int W = D / 32, NG = W / WPG;
  grid_wait();
  grid_go();  // the attention of these tokens may get ready
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int half = (int)blockIdx.x * 4 + (threadIdx.x >> 5), h = blockIdx.y;
  if (half >= n_halves) return;
  const int b = half_seq[half];
  const int len = S.kv_len[b], q0 = S.q_start[b], n = S.q_start[b + 1] - q0, first = len - n;
  const int tok0 = (first / 8 + half - half_start[b]) * 8, pos = tok0 + r;
  const bool valid = pos >= first && pos < len;
  Eight<T> k[W], v[W];
  if (valid) {
    const int64_t row = (int64_t)(pos - first) + (in.packed ? q0 : 0);
    const int64_t at = (in.packed ? 0 : b * in.sb) + row * in.st + h * in.sh + 8 * c;
#pragma unroll
    for (int w = 0; w < W; ++w) k[w].load(static_cast<const T*>(in.k) + at + 32 * w, in.vec != 0);
#pragma unroll
    for (int w = 0; w < W; ++w) v[w].load(static_cast<const T*>(in.v) + at + 32 * w, in.vec != 0);
  } else {
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int i = 0; i < Eight<T>::N; ++i) k[w].r[i] = v[w].r[i] = 0;
  }
  const int64_t page = page_of(L, S.rows[b], tok0, &tc::g_kvc_device_error);
  if (page < 0) return;
  uint8_t* unit = pool + unit_off<D>(L, page, h, tok0);
  const int t = pos & 15, p = (tok0 >> 3) & 1;
  uint32_t word[W];
  __half2 par[NG];

  quantise<T, W, WPG>(k, word, par);
  if (valid) {
    store_words<W>(unit + k_chunk<D>(t, c), word);
    if (c == 0)
#pragma unroll
      for (int g = 0; g < NG; ++g) reinterpret_cast<__half2*>(unit + kp_base(D))[t * NG + g] = par[g];
  }

  quantise<T, W, WPG>(v, word, par);
  if (valid && c == 0)
#pragma unroll
    for (int g = 0; g < NG; ++g) reinterpret_cast<__half2*>(unit + vp_base(D, NG))[t * NG + g] = par[g];
  const int cc = r >> 1, odd = r & 1;
  if (tok0 >= first && tok0 + 8 <= len) {
    // token pairs are neighbouring lanes (lane ^ 4): the even token's lane
    // takes features 4 (2 c) .. of both, the odd one's the next four
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? word[w] & 0xFFFFu : word[w] >> 16, 4);
      word[w] = odd ? got | (word[w] & 0xFFFF0000u) : (word[w] & 0xFFFFu) | got << 16;
    }
    store_words<W>(unit + v_chunk<D>(p, (2 * c + odd) * 4 + cc), word);
  } else if (valid) {
    // other tokens of the half keep their codes: two bytes hold four features
    // of one token
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        *reinterpret_cast<uint16_t*>(unit + v_chunk<D>(p, (2 * c + j) * 4 + cc) + w * 4 + odd * 2) =
            (uint16_t)(word[w] >> (16 * j));
  }
}

template <int W>
__device__ __forceinline__ void load_words(const uint8_t* src, uint32_t (&word)[W]) {
  if constexpr (W == 4) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(src));
    word[0] = a.x, word[1] = a.y, word[2] = a.z, word[3] = a.w;
  } else {
    const uint2 a = __ldg(reinterpret_cast<const uint2*>(src));
    word[0] = a.x, word[1] = a.y;
  }
}

// Dense (layers, n_kv, t1 - t0, D) K and V of tokens [t0, t1) of one sequence.
template <typename T, int D, int WPG>
__global__ void __launch_bounds__(128) kv4_read_kernel(Layout L, const uint8_t* pool, int64_t layer_bytes, int row,
                                                       int t0, int t1, int n_halves, T* __restrict__ ko,
                                                       T* __restrict__ vo) {
  constexpr int W = D / 32, NG = W / WPG;
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int half = (int)blockIdx.x * 4 + (threadIdx.x >> 5), h = blockIdx.y, layer = blockIdx.z;
  if (half >= n_halves) return;
  const int tok0 = (t0 / 8 + half) * 8, pos = tok0 + r, t = pos & 15;
  const int64_t page = page_of(L, row, tok0, &tc::g_kvc_device_error);
  if (page < 0) return;
  const uint8_t* unit = pool + layer * layer_bytes + unit_off<D>(L, page, h, tok0);

  const int odd = r & 1, p = (tok0 >> 3) & 1;
  uint32_t word[2][W];  // K's and V's
  __half2 par[2][NG];
  load_words<W>(unit + k_chunk<D>(t, c), word[0]);
  load_words<W>(unit + v_chunk<D>(p, (2 * c + odd) * 4 + (r >> 1)), word[1]);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    par[0][g] = reinterpret_cast<const __half2*>(unit + kp_base(D))[t * NG + g];
    par[1][g] = reinterpret_cast<const __half2*>(unit + vp_base(D, NG))[t * NG + g];
  }
#pragma unroll
  for (int w = 0; w < W; ++w) {  // the write's exchange again: it is its own inverse
    const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? word[1][w] & 0xFFFFu : word[1][w] >> 16, 4);
    word[1][w] = odd ? got | (word[1][w] & 0xFFFF0000u) : (word[1][w] & 0xFFFFu) | got << 16;
  }
  if (pos < t0 || pos >= t1) return;
  const int64_t at = (((int64_t)layer * L.n_kv + h) * (int64_t)(t1 - t0) + (pos - t0)) * D + 8 * c;
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    T* dst = (v ? vo : ko) + at;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float s = __low2float(par[v][w / WPG]), z = __high2float(par[v][w / WPG]);
      // nibbles i and i + 4 of a word, elements i ^ 1 and (i ^ 1) + 4, as float16
      // c - 8 (exact), then zero + scale * q in float32
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t y = word[v][w] >> (i & 2 ? 8 : 0);
        const float2 q = i & 1 ? __half22float2(centred_hi(y)) : __half22float2(centred_lo(y));
        x[i ^ 1] = fmaf(q.x, s, z);
        x[(i ^ 1) + 4] = fmaf(q.y, s, z);
      }
      store8(dst + 32 * w, x);
    }
  }
}

// ---- page copies ------------------------------------------------------------

// Page pairs of a launch, by value: no staging buffer to keep alive.  Few pairs
// (a fork's) go in a small one, since a launch copies its parameters.
constexpr int kPairs = 1024, kFewPairs = 32;
constexpr int kCopyBytes = 16384;

template <int N>
struct CopyPairs {
  int32_t src[N], dst[N];
};

// Bound by memory: four 16-byte loads in flight a thread, 16 KB a block; 300
// pages of 32 KB in each of 32 pools take 100 us (6.3 TB/s read and written).
template <typename V, int N>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CellPtrsMut pools,
                                                         const __grid_constant__ CopyPairs<N> pairs, int64_t page_bytes,
                                                         int parts) {
  const int pair = blockIdx.x / parts, part = blockIdx.x % parts;
  uint8_t* base = static_cast<uint8_t*>(pools.p[blockIdx.y]);
  const int64_t off = (int64_t)part * kCopyBytes;
  const int n = (int)((page_bytes - off < kCopyBytes ? page_bytes - off : kCopyBytes) / (int64_t)sizeof(V));
  const V* src = reinterpret_cast<const V*>(base + pairs.src[pair] * page_bytes + off);
  V* dst = reinterpret_cast<V*>(base + pairs.dst[pair] * page_bytes + off);
  for (int i = threadIdx.x; i < n; i += 4 * 256) {
    V v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j * 256 < n) v[j] = src[i + j * 256];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j * 256 < n) dst[i + j * 256] = v[j];
  }
}

}  // namespace

int check_layout(const kvc_kv4_layout* l, const char* what) {
  const std::string w(what);
  if (!l || !l->table) return fail(KVC_ERR_ARG, w + ": NULL layout or table");
  if (l->head_dim != 64 && l->head_dim != 128) return fail(KVC_ERR_SHAPE, w + ": head_dim must be 64 or 128");
  if (l->page_size < 16 || l->page_size > 256 || (l->page_size & (l->page_size - 1)))
    return fail(KVC_ERR_SHAPE, w + ": page_size must be 16, 32, 64, 128 or 256");
  const int g = l->group_size;
  if ((g != 32 && g != 64 && g != 128) || l->head_dim % g)
    return fail(KVC_ERR_SHAPE, w + ": group_size must be 32, 64 or 128 and divide head_dim");
  if (l->n_kv < 1 || l->n_pages < 1 || l->n_pages > INT32_MAX || l->table_stride < 1)
    return fail(KVC_ERR_SHAPE, w + ": bad layout sizes");
  return KVC_OK;
}

Layout to_layout(const kvc_kv4_layout* l) {
  int log2 = 4;
  while ((1 << log2) < l->page_size) ++log2;
  return Layout{l->n_pages, l->n_kv, log2, l->head_dim / l->group_size, l->table, l->table_stride};
}

}  // namespace kv4
}  // namespace kvc

using namespace kvc;
using namespace kvc::kv4;

extern "C" int64_t kvc_kv4_page_bytes(int n_kv, int head_dim, int page_size, int group_size) {
  if (n_kv < 1 || head_dim < 1 || page_size < 16 || group_size < 1) return 0;
  return (int64_t)n_kv * (page_size / kUnit) * unit_bytes(head_dim, head_dim / group_size);
}

extern "C" int kvc_kv4_write(const kvc_kv4_layout* layout, const kvc_kv4_step* step, void* pool, const void* k,
                             const void* v, int dtype, int64_t seq_stride, int64_t token_stride, int64_t head_stride,
                             int packed, void* stream) {
  if (int rc = check_layout(layout, "kvc_kv4_write")) return rc;
  if (!step || !pool) return fail(KVC_ERR_ARG, "kvc_kv4_write: NULL pointer");
  if (!dtype_ok(dtype)) return fail(KVC_ERR_DTYPE, "kvc_kv4_write: bad dtype");
  if (!aligned16(pool)) return fail(KVC_ERR_ALIGN, "kvc_kv4_write: pool not 16-byte aligned");
  if (step->n_halves < 0 || step->n_seqs < 0) return fail(KVC_ERR_SHAPE, "kvc_kv4_write: negative size");
  if (step->n_halves == 0) return KVC_OK;
  if (!k || !v || !step->rows || !step->kv_len || !step->q_start || !step->half_seq || !step->half_start)
    return fail(KVC_ERR_ARG, "kvc_kv4_write: NULL pointer");
  if (step->n_halves > INT32_MAX / 4 || layout->n_kv > 65535)
    return fail(KVC_ERR_SHAPE, "kvc_kv4_write: too many tokens or KV heads in one call");
  const dim3 grid((unsigned)ceil_div(step->n_halves, 4), (unsigned)layout->n_kv);
  const int64_t e = (int64_t)dtype_size(dtype);
  const bool vec = aligned16(k) && aligned16(v) && (seq_stride * e) % 16 == 0 && (token_stride * e) % 16 == 0 &&
                   (head_stride * e) % 16 == 0;
  const KvIn in{k, v, seq_stride, token_stride, head_stride, packed, vec};
  const Step s{step->n_seqs, step->rows, step->kv_len, step->q_start};
  const Layout L = to_layout(layout);
  int rc = KVC_OK;
#define KVC_F(D, WPG)                                                                                               \
  KVC_DISPATCH_DTYPE(dtype, T,                                                                                      \
                     rc = launch_after("kv4_write_kernel", kv4_write_kernel<T, D, WPG>, grid, 128, 0,               \
                                       static_cast<cudaStream_t>(stream), L, s, static_cast<uint8_t*>(pool), in,    \
                                       (int)step->n_halves, step->half_seq, step->half_start))
  KVC_KV4_DISPATCH(layout, KVC_F);
#undef KVC_F
  return rc;
}

extern "C" int kvc_kv4_read(const kvc_kv4_layout* layout, const void* pool, int64_t layer_bytes, int n_layers, int row,
                            int64_t t0, int64_t t1, int dtype, void* k_out, void* v_out, void* stream) {
  if (int rc = check_layout(layout, "kvc_kv4_read")) return rc;
  if (!pool || !k_out || !v_out) return fail(KVC_ERR_ARG, "kvc_kv4_read: NULL pointer");
  if (!dtype_ok(dtype)) return fail(KVC_ERR_DTYPE, "kvc_kv4_read: bad dtype");
  if (!aligned16(pool) || !aligned16(k_out) || !aligned16(v_out) || layer_bytes % 16)
    return fail(KVC_ERR_ALIGN, "kvc_kv4_read: pool, layers and outputs must be 16-byte aligned");
  if (n_layers < 0 || row < 0 || t0 < 0 || t1 < t0 || t1 > layout->table_stride * layout->page_size || t1 > INT32_MAX)
    return fail(KVC_ERR_SHAPE, "kvc_kv4_read: bad layers or token range");
  if (t0 == t1 || n_layers == 0) return KVC_OK;
  const int64_t halves = (t1 - 1) / 8 - t0 / 8 + 1;
  if (layout->n_kv > 65535 || n_layers > 65535) return fail(KVC_ERR_SHAPE, "kvc_kv4_read: too many layers or KV heads");
  const dim3 grid((unsigned)ceil_div(halves, 4), (unsigned)layout->n_kv, (unsigned)n_layers);
  const Layout L = to_layout(layout);
#define KVC_F(D, WPG)                                                                                        \
  KVC_DISPATCH_DTYPE(dtype, T,                                                                               \
                     (kv4_read_kernel<T, D, WPG><<<grid, 128, 0, static_cast<cudaStream_t>(stream)>>>(             \
                         L, static_cast<const uint8_t*>(pool), layer_bytes, row, (int)t0, (int)t1, (int)halves,    \
                         static_cast<T*>(k_out), static_cast<T*>(v_out))))
  KVC_KV4_DISPATCH(layout, KVC_F);
#undef KVC_F
  return check_launch("kv4_read_kernel");
}

extern "C" int kvc_copy_pages(int n_pools, void* const* pools, int64_t n_pages, int64_t page_bytes, int64_t n_pairs,
                              const int32_t* src, const int32_t* dst, void* stream) {
  if (n_pools < 0 || n_pools > KVC_MAX_CELLS || n_pages < 0 || page_bytes < 0 || n_pairs < 0)
    return fail(KVC_ERR_SHAPE, "kvc_copy_pages: bad sizes");
  if (n_pools == 0 || n_pairs == 0 || page_bytes == 0) return KVC_OK;
  if (!pools || !src || !dst) return fail(KVC_ERR_ARG, "kvc_copy_pages: NULL pointer");
  CellPtrsMut p{};
  bool a16 = page_bytes % 16 == 0, a4 = page_bytes % 4 == 0;
  for (int i = 0; i < n_pools; ++i) {
    if (!pools[i]) return fail(KVC_ERR_ARG, "kvc_copy_pages: NULL pool");
    p.p[i] = pools[i];
    a16 = a16 && aligned16(pools[i]);
    a4 = a4 && (reinterpret_cast<uintptr_t>(pools[i]) & 3u) == 0;
  }
  for (int64_t i = 0; i < n_pairs; ++i)
    if (src[i] < 0 || src[i] >= n_pages || dst[i] < 0 || dst[i] >= n_pages)
      return fail(KVC_ERR_SHAPE, "kvc_copy_pages: page out of range");
  const int64_t parts = ceil_div(page_bytes, kCopyBytes);
  if (parts > INT32_MAX / kPairs) return fail(KVC_ERR_SHAPE, "kvc_copy_pages: page too large");
  auto launch = [&](auto& pr, auto limit) {
    constexpr int N = decltype(limit)::value;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    for (int64_t at = 0; at < n_pairs; at += N) {
      const int n = (int)std::min<int64_t>(N, n_pairs - at);
      memcpy(pr.src, src + at, n * sizeof(int32_t));
      memcpy(pr.dst, dst + at, n * sizeof(int32_t));
      const dim3 grid((unsigned)(n * parts), (unsigned)n_pools);
      if (a16) copy_pages_kernel<uint4, N><<<grid, 256, 0, st>>>(p, pr, page_bytes, (int)parts);
      else if (a4) copy_pages_kernel<uint32_t, N><<<grid, 256, 0, st>>>(p, pr, page_bytes, (int)parts);
      else copy_pages_kernel<uint8_t, N><<<grid, 256, 0, st>>>(p, pr, page_bytes, (int)parts);
      if (int rc = check_launch("copy_pages_kernel")) return rc;
    }
    return (int)KVC_OK;
  };
  if (n_pairs <= kFewPairs) {
    CopyPairs<kFewPairs> pr;
    return launch(pr, std::integral_constant<int, kFewPairs>{});
  }
  CopyPairs<kPairs> pr;
  return launch(pr, std::integral_constant<int, kPairs>{});
}
