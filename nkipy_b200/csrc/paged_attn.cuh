// The forms of paged attention (k_paged_attn.cu chooses) and what they share.
#pragma once

#include "paged.cuh"

namespace nkb {
namespace pattn {

using Args = nkb_paged_attention_args;

// Keys that the last token of a sequence sees, as one run of n "virtual" keys:
// the first `ns` are keys 0 .. ns - 1 (the first tokens that stay visible), the
// others keys low, low + 1, ... up to the end.
struct Visible {
  int ns, low, n;
  __device__ __forceinline__ int key(int v) const { return v < ns ? v : v - ns + low; }
};
// token at `pos`; `cap` positions have a place in the page table
__device__ __forceinline__ Visible visible(int64_t pos, int64_t cap, int64_t window, int64_t sinks) {
  Visible r;
  const int64_t end = max((int64_t)0, min(pos + 1, cap));
  const int64_t low = window > 0 ? min(max((int64_t)0, pos - window + 1), end) : 0;
  r.ns = (int)min(sinks, low);
  r.low = (int)low;
  r.n = r.ns + (int)(end - low);
  return r;
}

// ---- work split evenly over the resident CTAs --------------------------------
// The key blocks of all units, one run of `total`, are cut into equal shares.
// CTAs that share the blocks: none of them is left without one
__host__ __device__ __forceinline__ int workers(int64_t total, int ctas) { return total < ctas ? (int)total : ctas; }
// first block of CTA c's share
__device__ __forceinline__ int64_t share(int64_t total, int c, int ctas) { return total * c / ctas; }
// CTA whose share holds block f
__device__ __forceinline__ int owner(int64_t total, int64_t f, int ctas) {
  int c = (int)(f * ctas / total);
  while (share(total, c + 1, ctas) <= f) ++c;
  while (share(total, c, ctas) > f) --c;
  return c;
}
// The partials of a unit whose blocks are [first, first + nb): the slots they
// lie in.  A CTA's first segment has slot 2c, a later one that goes on in the
// next CTA 2c + 1; a unit that one CTA holds whole is written out at once, or,
// where everything is kept for a later join, lies in slot 2 * max_ctas + unit.
struct Parts {
  int n, c0, s0;
  __device__ __forceinline__ int slot(int i) const { return i ? 2 * (c0 + i) : s0; }
};
__device__ __forceinline__ Parts parts_of(int64_t total, int64_t first, int64_t nb, int max_ctas, int64_t unit) {
  const int ctas = workers(total, max_ctas), c0 = owner(total, first, ctas), c1 = owner(total, first + nb - 1, ctas);
  Parts p;
  p.n = c1 - c0 + 1;
  p.c0 = c0;
  p.s0 = c0 == c1 ? 2 * max_ctas + (int)unit : 2 * c0 + (share(total, c0, ctas) != first);
  return p;
}

// 2^x on the special-function unit (relative error about 2^-22; -inf -> 0)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two values rounded to the 16-bit type
template <class T>
__device__ __forceinline__ uint32_t pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack<__half>(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&h);
}

// rows of 16-byte pieces: every stride and base that a vector or TMA access needs
inline bool aligned16(const Args &a) {
  const int64_t s[] = {a.q_token, a.q_head, a.out_token, a.out_head, a.k_page, a.k_slot, a.k_cache_head,
                       a.v_page, a.v_slot, a.v_cache_head, a.head_dim};
  for (int64_t x : s)
    if (x < 0 || x % 8) return false;
  const void *p[] = {a.q, a.out, a.k_cache, a.v_cache};
  for (const void *x : p)
    if (reinterpret_cast<uintptr_t>(x) & 15) return false;
  return true;
}

// single tokens (k_paged_decode.cu)
size_t decode_workspace(const Args &a, int device);
int decode_run(const Args &a, cudaStream_t st, int device);

// several tokens per sequence (k_paged_tile.cu)
bool tile_form(const Args &a);     // by the sizes
bool tile_strides(const Args &a);  // whether TMA can describe the operands
size_t tile_workspace(const Args &a, int device);
int tile_run(const Args &a, cudaStream_t st, int device);
int tile_read_and_clear_error(int *flag);

}  // namespace pattn
}  // namespace nkb
