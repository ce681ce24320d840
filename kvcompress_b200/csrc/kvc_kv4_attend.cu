// Attention over the pages of the 4-bit KV cache.
//
// softmax(scale q k^T) v with one pass over the tokens: running maximum m,
// sum l and accumulator o, rescaled by exp(m_old - m_new) when m grows; all in
// float32.  A warp per query and head; each lane holds D / 32 features.
#include "kvc_kv4.cuh"
#include "kvc_tc.cuh"

namespace kvc {

int kv4_attend_read_device_error(int* out) {
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

struct Qkv {
  const void* q;
  void* out;
  int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh;
  int packed, dtype, n_q, causal;
  float scale;
};

// Code 0..15 of feature x of token t (0..15) in a unit.
template <int D>
__device__ __forceinline__ int k_code(const uint8_t* unit, int t, int x) {
  const uint8_t b = unit[k_chunk<D>(t, (x & 31) >> 3) + (x >> 5) * 4 + ((x & 7) >> 1)];
  return x & 1 ? b & 15 : b >> 4;
}
template <int D>
__device__ __forceinline__ int v_code(const uint8_t* unit, int t, int x) {
  const int r = (x & 31) >> 2, c = (t & 7) >> 1;
  const uint8_t b = unit[v_chunk<D>(t >> 3, r * 4 + c) + (x >> 5) * 4 + (t & 1) * 2 + ((x & 3) >> 1)];
  return x & 1 ? b & 15 : b >> 4;
}

template <int D>
__global__ void __launch_bounds__(128) attend_simple_kernel(Layout L, Step S, const uint8_t* pool, Qkv a) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31, head = blockIdx.y * 4 + (threadIdx.x >> 5), tok = blockIdx.x;
  if (head >= a.n_q) return;
  int b = 0;
  while (b + 1 < S.n_seqs && S.q_start[b + 1] <= tok) ++b;
  const int q0 = S.q_start[b], n = S.q_start[b + 1] - q0, j = tok - q0, len = S.kv_len[b];
  const int seen = a.causal ? len - n + 1 + j : len, h = head / (a.n_q / L.n_kv), gw = 32 * E / L.groups;
  const int64_t row = a.packed ? tok : j;
  const int64_t qo = (a.packed ? 0 : b * a.q_sb) + row * a.q_st + head * a.q_sh;
  float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) q[e] = load_dt(a.q, qo + e * 32 + lane, a.dtype), o[e] = 0.0f;
  for (int t = 0; t < seen; ++t) {
    const int64_t page = page_of(L, S.rows[b], t, &tc::g_kvc_device_error);
    if (page < 0) continue;
    const uint8_t* unit = pool + unit_off<D>(L, page, h, t);
    const __half2* kp = reinterpret_cast<const __half2*>(unit + kp_base(D)) + (t & 15) * L.groups;
    const __half2* vp = reinterpret_cast<const __half2*>(unit + vp_base(D, L.groups)) + (t & 15) * L.groups;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int x = e * 32 + lane;
      const float2 p = __half22float2(kp[x / gw]);
      s += q[e] * fmaf((float)(k_code<D>(unit, t & 15, x) - 8), p.x, p.y);
    }
#pragma unroll
    for (int i = 16; i; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    s *= a.scale;
    const float m2 = fmaxf(m, s), f = __expf(m - m2), w = __expf(s - m2);
    l = l * f + w;
    m = m2;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int x = e * 32 + lane;
      const float2 p = __half22float2(vp[x / gw]);
      o[e] = o[e] * f + w * fmaf((float)(v_code<D>(unit, t & 15, x) - 8), p.x, p.y);
    }
  }
  const int64_t oo = (a.packed ? 0 : b * a.o_sb) + row * a.o_st + head * a.o_sh;
#pragma unroll
  for (int e = 0; e < E; ++e) store_dt(a.out, oo + e * 32 + lane, seen > 0 ? o[e] / l : 0.0f, a.dtype);
}

}  // namespace
}  // namespace kv4
}  // namespace kvc

using namespace kvc;
using namespace kvc::kv4;

extern "C" size_t kvc_kv4_attend_workspace_bytes(const kvc_kv4_layout*, const kvc_kv4_step*, const kvc_kv4_split*, int) {
  return 0;
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
  if (n_q < 1 || n_q % layout->n_kv) return fail(KVC_ERR_SHAPE, "kvc_kv4_attend: n_q must be a multiple of n_kv");
  if (step->n_tokens == 0) return KVC_OK;
  const Step s{step->n_seqs, step->rows, step->kv_len, step->q_start};
  const Qkv a{q, out, q_seq_stride, q_token_stride, q_head_stride, o_seq_stride, o_token_stride, o_head_stride,
              packed, dtype, n_q, causal, scale};
  const dim3 grid((unsigned)step->n_tokens, (unsigned)ceil_div(n_q, 4));
  const Layout L = to_layout(layout);
  if (layout->head_dim == 64)
    attend_simple_kernel<64><<<grid, 128, 0, static_cast<cudaStream_t>(stream)>>>(L, s, static_cast<const uint8_t*>(pool), a);
  else
    attend_simple_kernel<128><<<grid, 128, 0, static_cast<cudaStream_t>(stream)>>>(L, s, static_cast<const uint8_t*>(pool), a);
  return check_launch("attend_simple_kernel");
}
