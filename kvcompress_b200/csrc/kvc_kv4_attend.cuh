// What the attention kernels of the 4-bit KV cache share.
#pragma once

#include "kvc_kv4.cuh"
#include "kvc_tma.cuh"

namespace kvc {
namespace kv4 {

constexpr int kGridZ = 65535;  // a grid's largest extent in z: more column tiles or items are several launches
constexpr float kLog2e = 1.4426950408889634f;
// log2 units a logit may exceed its row's reference by: raising costs a pass over
// the accumulators, and float16 weights have room for 2^15 (4 instead of 8: 5% more
// time for the attention of many queries)
constexpr float kRaise = 8.0f;

struct Qkv {
  const void* q;
  void* out;
  int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh;  // element strides of a sequence, a token, a head
  int packed, dtype, n_q, causal;
  float scale;
};

struct Split {
  const int4* items;          // sequence, first and last + 1 token, table row
  const int32_t *item_start;  // of each sequence
  const int32_t *block_start; // items of each block (kernel for few columns)
  int max_items;
};

// Partial results of an item: o (unnormalised) and (m, l) of each of its
// sequence's columns, [item][KV head][column].
struct Partial {
  float* o;
  float2* ml;
  int64_t cols;  // columns of an item and KV head
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  uint32_t r;
  memcpy(&r, &h, 4);
  return r;
}
__device__ __forceinline__ float2 unpack_half2(uint32_t r) {
  __half2 h;
  memcpy(&h, &r, 4);
  return __half22float2(h);
}

template <int W>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[W]) {
  if constexpr (W == 4)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(addr));
  else if constexpr (W == 2)
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  else
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}

// Tokens that query j of n sees of len.
__device__ __forceinline__ int visible(int causal, int len, int n, int j) {
  return causal ? max(0, len - n + 1 + j) : len;
}

// Attention of many 16-bit queries (kvc_kv4_prefill.cu); its blocks take 256
// rows (part.cols of them to a sequence and KV head).
int launch_prefill(const kvc_kv4_layout* l, const Step& S, const Split& P, const uint8_t* pool, const Qkv& a,
                   const Partial& part, int64_t n_items, cudaStream_t st);
inline int64_t prefill_tiles(int64_t rows) { return ceil_div(rows, 256); }
int prefill_read_device_error(int* out);

}  // namespace kv4
}  // namespace kvc
