// Shared by the paged-cache kernels: which sequence and position a new token
// has, and where a position's row lies in the pages.
#pragma once

#include <cstring>

#include "common.cuh"

namespace nkb {
namespace paged {

// Pages of one cache operand as the kernels address them (element strides).
struct Pages {
  int64_t page, slot, head;
};

// page id -> valid in a cache of `pages` pages
__device__ __forceinline__ bool page_ok(int id, int64_t pages) { return id >= 0 && id < pages; }

// Sequence of token t, found by every thread of the block together: each
// thread looks at some of the sequences, so the search costs one load latency
// whatever their number.  -1 when no sequence owns the token.  `slot` is one
// shared int; all threads return the same value.
__device__ __forceinline__ int block_find_seq(const int32_t *q_start, int seqs, int t, int *slot) {
  if (!q_start) return t < seqs ? t : -1;
  if (threadIdx.x == 0) *slot = -1;
  __syncthreads();
  for (int b = threadIdx.x; b < seqs; b += blockDim.x)
    if (q_start[b] <= t && t < q_start[b + 1]) *slot = b;
  __syncthreads();
  return *slot;
}

template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }

inline bool float_dtype(int64_t dt) { return dt == NKB_F32 || dt == NKB_BF16 || dt == NKB_F16; }

// f(T{}) with the element type of `dt`
template <class F>
int with_dtype(int64_t dt, F &&f) {
  if (dt == NKB_F32) return f(float{});
  if (dt == NKB_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}

// The argument struct of a plan step: its pointers first, then 8-byte integers
// (and doubles, from the step's floats).  ints[0] has a bit for each pointer
// that is given, in order; ptrs is NULL while a plan is checked.
template <class A>
int step_args(const Step &s, void *const *ptrs, int n_ptrs, int n_ints, const char *what, A *a) {
  static_assert(sizeof(void *) == 8 && sizeof(int64_t) == 8, "8-byte fields");
  const int n_floats = (int)(sizeof(A) / 8) - n_ptrs - n_ints;
  auto bad = [&]() { return fail(NKB_ERR_PLAN, std::string(what) + ": bad parameters"); };
  if ((int)s.ints.size() != n_ints + 1 || (int)s.floats.size() != n_floats) return bad();
  if (s.ints[0] < 0 || s.ints[0] >> n_ptrs) return bad();
  char *at = reinterpret_cast<char *>(a);
  size_t next = 0;
  for (int i = 0; i < n_ptrs; ++i) {
    void *p = nullptr;
    if (s.ints[0] >> i & 1) {
      if (next >= s.buf_ids.size()) return bad();
      p = ptrs ? ptrs[next] : reinterpret_cast<void *>(16);  // any that is not NULL and aligned
      ++next;
    }
    memcpy(at + 8 * i, &p, 8);
  }
  if (next != s.buf_ids.size()) return bad();
  for (int i = 0; i < n_ints; ++i) memcpy(at + 8 * (n_ptrs + i), &s.ints[1 + i], 8);
  for (int i = 0; i < n_floats; ++i) {
    const double f = s.floats[i];
    memcpy(at + 8 * (n_ptrs + n_ints + i), &f, 8);
  }
  return NKB_OK;
}

// Positions that a page table or a prefix may hold: rounded up to a block of keys they stay in 32 bits.
constexpr int64_t MAX_POSITIONS = (int64_t(1) << 31) - 256;

// What every call on a paged cache requires of its sizes (names for messages).
inline int check_cache(const char *what, int64_t tokens, int64_t seqs, int64_t kv_heads, int64_t head_dim, int64_t pages,
                       int64_t page_size, int64_t width, int64_t table_stride) {
  auto bad = [&](const char *m) { return fail(NKB_ERR_INVALID, std::string(what) + ": " + m); };
  if (tokens < 0 || seqs < 0 || tokens > INT32_MAX || seqs > INT32_MAX) return bad("tokens or sequences out of range");
  if (kv_heads < 1 || head_dim < 1 || kv_heads > 65535) return bad("kv_heads or head_dim out of range");
  if (pages < 0 || pages > INT32_MAX || page_size < 1 || page_size > INT32_MAX) return bad("pages or page_size out of range");
  if (width < 0 || table_stride < 0 || (seqs > 1 && table_stride < width)) return bad("page table rows overlap");
  if (width > MAX_POSITIONS / page_size) return bad("page table holds more than 2^31 - 256 positions");
  return NKB_OK;
}

}  // namespace paged
}  // namespace nkb
