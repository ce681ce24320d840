// Paged 4-bit KV cache: the layout of its pages and the descriptors that the
// kernels take.
//
// A layer's pool is (n_pages, n_kv, page_size / 16, unit_bytes).  A unit holds
// 16 tokens of one head:
//   [K codes 8 d][V codes 8 d][K parameters 64 groups][V parameters 64 groups]
// so that any run of a page's units is one contiguous, 16-byte aligned copy.
// x = zero + scale * (code - 8) with code in 0..15; parameters are half2
// (scale, zero), [token][group].  Code words hold 8 elements, the first of
// each byte in its high nibble.
//
// The codes lie as the tensor-core fragments want them (m16n8k16, A operand),
// so that a lane's 16-byte load is its fragment without any shuffles:
//  * K (row = token, k = feature): token t's row of d/2 bytes is four chunks
//    of d/8 bytes, chunk c for lanes with lane % 4 == c; word w of chunk c is
//    features 32 w + 8 c + 0..7, so that two k-steps cover one aligned run of
//    32 features and a quantisation group of 32 or more never splits a k-step.
//  * V (row = feature, k = token): word u of lane l = 4 r + c, token pair block
//    p (tokens 8 p + 2 c and 8 p + 2 c + 1): features 32 u + 4 r + 0..3 of the
//    first token in its low half, of the second in its high half.
#pragma once

#include <atomic>

#include "kvc_common.cuh"

namespace kvc {
namespace kv4 {

constexpr int kUnit = 16;               // tokens of a unit
constexpr float kLimit = 65024.0f;      // held magnitudes: zero + 15 scale stays below float16's largest value

__host__ __device__ constexpr int unit_bytes(int d, int groups) { return 16 * d + 128 * groups; }
__host__ __device__ constexpr int v_base(int d) { return 8 * d; }
__host__ __device__ constexpr int kp_base(int d) { return 16 * d; }
__host__ __device__ constexpr int vp_base(int d, int groups) { return 16 * d + 64 * groups; }

// Byte of K's chunk c of token t (0..15), from the unit's start.
template <int D>
__device__ __forceinline__ int k_chunk(int t, int c) {
  return t * (D / 2) + c * (D / 8);
}
// Byte of V's words (u = 0, 1, ...) of lane l and token pair block p.
template <int D>
__device__ __forceinline__ int v_chunk(int p, int l) {
  static_assert(D == 64 || D == 128, "head_dim");
  return v_base(D) + (D == 128 ? p * 512 + l * 16 : l * 16 + p * 8);
}

struct Layout {
  int64_t n_pages;
  int n_kv, page_log2, groups;
  const int32_t* table;    // (rows, table_stride) page ids
  int64_t table_stride;
};

struct Step {
  int n_seqs;
  const int32_t* rows;     // table row of each sequence
  const int32_t* kv_len;   // cached tokens, the step's own among them
  const int32_t* q_start;  // n_seqs + 1: the step's tokens of each sequence
};

// Page of token `pos` of table row `row`; -1 (and the error word) for an entry
// that is no page of the pool.
__device__ __forceinline__ int64_t page_of(const Layout& L, int64_t row, int64_t pos, int* error) {
  const int64_t p = L.table[row * L.table_stride + (pos >> L.page_log2)];
  if (p < 0 || p >= L.n_pages) {
    atomicCAS(error, 0, 401);
    return -1;
  }
  return p;
}

// Byte offset of the unit that holds token `pos` of head h on page p.
template <int D>
__device__ __forceinline__ int64_t unit_off(const Layout& L, int64_t p, int h, int64_t pos) {
  const int per_page = 1 << (L.page_log2 - 4);
  return ((p * L.n_kv + h) * per_page + ((pos >> 4) & (per_page - 1))) * (int64_t)unit_bytes(D, L.groups);
}

// A pair of codes as float16 c - 8: nibble 0 of each half from 1024 + c, nibble
// 1 from 1024 + 16 c.  Both steps are exact.
__device__ __forceinline__ __half2 centred_lo(uint32_t w) {
  uint32_t x = (w & 0x000F000Fu) | 0x64006400u, off = 0x64086408u;  // 1032
  __half2 h, o;
  memcpy(&h, &x, 4);
  memcpy(&o, &off, 4);
  return __hsub2(h, o);
}
__device__ __forceinline__ __half2 centred_hi(uint32_t w) {
  uint32_t x = (w & 0x00F000F0u) | 0x64006400u, scale = 0x2C002C00u, off = 0xD480D480u;  // 1 / 16, -72
  __half2 h, s, o;
  memcpy(&h, &x, 4);
  memcpy(&s, &scale, 4);
  memcpy(&o, &off, 4);
  return __hfma2(h, s, o);
}
// Programmatic launches: a kernel launched with launch_after may start while
// the previous one of its stream runs; grid_wait returns when that one is
// complete and its writes are visible.  Every thread comes by it, before it
// ends too, so that a kernel's end is also the end of those before it.  Only the
// step's and the split's arrays and the page table are read earlier.  So whatever
// writes an entry that a kernel here will read must not be the very kernel in front
// of it: a copy, or an ordinary kernel, has to lie between them in the stream.  The
// arrays are written by copies; the table is updated by a kernel, with the copy of a
// step's arrays behind it.  grid_go lets the next such kernel start (its grid_wait still waits
// for this grid's end); it comes after grid_wait, so that no more than two
// kernels are under way.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename K, typename... A>
int launch_after(const char* what, K kernel, dim3 grid, unsigned threads, size_t smem, cudaStream_t st, const A&... args) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return fail(KVC_ERR_LAUNCH, std::string(what) + ": " + cudaGetErrorString(e));
  return check_launch(what);
}

// Allow a kernel `bytes` of dynamic shared memory, once for each device (`done`
// is the kernel's own: a bit a device).
template <typename K>
int allow_shared(const char* what, K kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev >= 0 && dev < 64 ? uint64_t(1) << dev : 0;
  if (e == cudaSuccess && (done.load(std::memory_order_relaxed) & bit)) return KVC_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(KVC_ERR_LAUNCH, std::string(what) + ": " + cudaGetErrorString(e));
  done.fetch_or(bit, std::memory_order_relaxed);
  return KVC_OK;
}

// Host side: argument checks shared by the entry points.
int check_layout(const kvc_kv4_layout* l, const char* what);
Layout to_layout(const kvc_kv4_layout* l);
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace kv4
}  // namespace kvc

// F(D, words of 32 features a quantisation group) for the layout.
#define KVC_KV4_DISPATCH(l, F)                        \
  do {                                                \
    if ((l)->head_dim == 64) {                        \
      if ((l)->group_size == 32) F(64, 1);            \
      else F(64, 2);                                  \
    } else {                                          \
      if ((l)->group_size == 32) F(128, 1);           \
      else if ((l)->group_size == 64) F(128, 2);      \
      else F(128, 4);                                 \
    }                                                 \
  } while (0)
