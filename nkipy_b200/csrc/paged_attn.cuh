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

}  // namespace pattn
}  // namespace nkb
