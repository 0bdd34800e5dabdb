// The forms of paged attention (k_paged_attn.cu chooses) and what they share.
#pragma once

#include "paged.cuh"

namespace nkb {
namespace pattn {

using Args = nkb_paged_attention_args;
constexpr double LOG2E = 1.4426950408889634;

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
// (Few instructions, and few divisions among them: in calls of a few microseconds
// each of these steps is run once, from memory.)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}
struct Split {
  int64_t total, each;  // blocks; of a share, and one more for the first `more` CTAs
  int ctas, more;       // CTAs that share: none of them is left without a block
  __device__ __forceinline__ Split(int64_t blocks, int max_ctas)
      : total(blocks), ctas(blocks < max_ctas ? max(1, (int)blocks) : max_ctas) {
    each = quotient(total, ctas);
    more = (int)(total - each * ctas);
  }
  // first block of CTA c's share
  __device__ __forceinline__ int64_t first(int c) const { return each * c + min(c, more); }
  // CTA whose share holds block f
  __device__ __forceinline__ int owner(int64_t f) const {
    const int64_t longer = (each + 1) * more;
    return (int)(f < longer ? quotient(f, each + 1) : more + quotient(f - longer, each));
  }
};
// The partials of a unit whose blocks are [first, first + nb): the slots they
// lie in.  A CTA's first segment has slot 2c, a later one that goes on in the
// next CTA 2c + 1; a unit that one CTA holds whole is written out at once, or,
// where everything is kept for a later join, lies in slot 2 * max_ctas + unit.
struct Parts {
  int n, c0, s0;
  __device__ __forceinline__ int slot(int i) const { return i ? 2 * (c0 + i) : s0; }
};
__device__ __forceinline__ Parts parts_of(const Split &split, int64_t first, int64_t nb, int max_ctas, int64_t unit) {
  const int c0 = split.owner(first), c1 = split.owner(first + nb - 1);
  Parts p;
  p.n = c1 - c0 + 1;
  p.c0 = c0;
  p.s0 = c0 == c1 ? 2 * max_ctas + (int)unit : 2 * c0 + (split.first(c0) != first);
  return p;
}

// One partial of a row: where its four outputs and its (max, sum) lie.
struct Partial {
  const float *o, *ml;
};
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

// Running maxima may pass over NaN, which is then in the sum: a part with a maximum of -inf
// has seen nothing (its sum and outputs are 0) or nothing but NaN (its sum is NaN).
// `top` as the base of exponentials: 0 where nothing has been seen.
__device__ __forceinline__ float base_of(float top) { return top == -INFINITY ? 0.f : top; }
// 1 / sum; 0 for a row that sees nothing, NaN for NaN
__device__ __forceinline__ float inverse(float l) { return l > 0.f ? 1.f / l : l; }

// Four outputs of a row, joined from partials that are read U at a time.
template <int U>
struct Joined {
  float m = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
  template <class At>
  __device__ __forceinline__ void add(int n, At at) {
    add_from(
        n, [&](int j) { return __ldcg(reinterpret_cast<const float2 *>(at(j).ml)); },
        [&](int j) { return __ldcg(reinterpret_cast<const float4 *>(at(j).o)); });
  }
  template <class Ml, class Out>
  __device__ __forceinline__ void add_from(int n, Ml ml_at, Out o_at) {
    for (int j0 = 0; j0 < n; j0 += U) {
      float2 ml[U];
      float4 y[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        ml[j] = make_float2(-INFINITY, 0.f);
        y[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (j0 + j >= n) continue;
        ml[j] = ml_at(j0 + j);
        y[j] = o_at(j0 + j);
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < U; ++j) top = fmaxf(top, ml[j].x);
      if (top == -INFINITY) {  // nothing seen so far, or NaN
#pragma unroll
        for (int j = 0; j < U; ++j) l += ml[j].y;
        continue;
      }
      const float f = ex2(m - top);
      l *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] *= f;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const float g = ex2(ml[j].x - top);
        l += ml[j].y * g;
        x[0] += y[j].x * g;
        x[1] += y[j].y * g;
        x[2] += y[j].z * g;
        x[3] += y[j].w * g;
      }
      m = top;
    }
  }
  template <class T>
  __device__ __forceinline__ void store(T *p) const {
    const float inv = inverse(l);
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack<T>(x[0] * inv, x[1] * inv), pack<T>(x[2] * inv, x[3] * inv));
  }
};

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

// ---- single tokens (k_paged_decode.cu) -------------------------------------
namespace single {

constexpr int THREADS = 128, WARPS = 4, ROWS = 16;

template <int DP>
struct Shape {
  static constexpr int WN = DP == 128 ? 16 : 32;       // keys per warp and stage
  static constexpr int BK = WARPS * WN;                // keys per block
  static constexpr int TILE = WN * DP * 2;             // bytes of K (or V) per stage
  static constexpr int STAGES = 3;
  static constexpr int RING = STAGES * 2 * TILE;       // per warp
  static constexpr int QBUF = ROWS * DP * 2;           // Q of one segment: there are as many as stages
  static constexpr int SMEM = STAGES * QBUF + WARPS * RING + WARPS * ROWS * 8;
  static_assert(ROWS * DP * 4 <= 2 * TILE, "a warp's outputs fit a stage");
  static constexpr int SLOT = ROWS * (DP + 2);         // floats of one partial: outputs, then max and sum
};

struct Params {
  Args a;
  int groups;  // 16-row groups of query heads per key head
  float scale_log2;
  float *ws;
  int ctas;
  bool keep;  // write every result as a partial (a prefix is joined to it)
};

__device__ __forceinline__ Visible visible_of(const Args &a, int b) {
  return visible((int64_t)a.kv_len[b] - 1, a.table_width * a.page_size, a.window, a.sinks);
}
// key blocks of sequence b (one at least: a sequence without keys has a row of zeros to write)
template <int BK>
__device__ __forceinline__ int blocks_of(const Args &a, int b) {
  return max(1, (visible_of(a, b).n + BK - 1) / BK);
}

// Sum of blocks_of over all sequences, and the first sequence whose blocks
// before and in it reach past `f` units of `per` (its own included): found by
// all threads of the block together.
struct Found {
  int64_t total;   // blocks of all sequences
  int seq;         // the sequence
  int64_t before;  // blocks of the sequences before it
};
template <int BK, class Want>
__device__ __forceinline__ Found find(const Args &a, Want want) {
  __shared__ int64_t s_warp[WARPS], s_before;
  __shared__ int s_seq;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, B = (int)a.seqs;
  Found r;
  r.total = 0;
  int64_t n = 0, first = 0;  // blocks of this thread's sequence, and before it
  auto chunk = [&](int base) {
    const int b = base + (int)threadIdx.x;
    n = b < B ? blocks_of<BK>(a, b) : 0;
    int64_t p = n;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, p, w);
      if (lane >= w) p += x;
    }
    if (base) __syncthreads();  // the sums of the chunk before are read
    if (lane == 31) s_warp[warp] = p;
    __syncthreads();
    first = r.total + p - n;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) first += s_warp[w];
      r.total += s_warp[w];
    }
    return b;
  };
  int b = 0;
  for (int base = 0; base < B; base += THREADS) b = chunk(base);
  if (B <= THREADS) {
    if (b < B && want(r.total, b, first, n)) {
      s_seq = b;
      s_before = first;
    }
  } else {  // the sum was for the total: once more
    const int64_t total = r.total;
    r.total = 0;
    __syncthreads();
    for (int base = 0; base < B; base += THREADS) {
      b = chunk(base);
      if (b < B && want(total, b, first, n)) {
        s_seq = b;
        s_before = first;
      }
    }
  }
  __syncthreads();
  r.seq = s_seq;
  r.before = s_before;
  return r;
}

}  // namespace single

// `keep`: every result stays a partial in the workspace
size_t decode_workspace(const Args &a, int device, bool keep);
int decode_params(const Args &a, int device, void *workspace, bool keep, single::Params *p);
int decode_launch(const single::Params &p, cudaStream_t st, int device, bool pdl);

// ---- several tokens per sequence, a shared prefix (k_paged_tile.cu) ---------
namespace several {

constexpr int BM = 128, BN = 128;

// a pair: up to 2 P tokens of one sequence
struct Pair {
  int seq;  // -1: the shared prefix, -2: tokens of no sequence
  int tok0, ntok, pos0;
};

struct Params {
  Args a;
  int G, P, page_shift, max_pairs, max_ctas;
  int own, prefix;  // list the sequences' own keys / the prefix
  int keep;         // write every unit as a partial
  int inside;       // each CTA of the tile kernel lists the pairs for itself
  int wide;         // rows of out start at 32-byte boundaries
  float scale_log2;
  int64_t *head;   // number of pairs, the pairs' first blocks (max_pairs + 1), the longest one's blocks
  int *next;       // the next unit that no CTA has, where whole units are handed out
  Pair *pairs;
  int *seq_pairs;  // first pair of each sequence (scheduler only)
  float *ws;
};

// The key blocks of a pair: `ns` from block 0 (first tokens), then [w0, w0 + n - ns).
struct Blocks {
  int end, low;  // keys below `end`, and from `low` (or below `sinks`) are seen by some row
  int ns, w0, n;
  __device__ __forceinline__ int block(int i) const { return i < ns ? i : w0 + i - ns; }
};
__device__ __forceinline__ Blocks blocks_of(const Params &p, const Pair &x) {
  Blocks r;
  if (x.seq < 0) {
    r.end = x.seq == -1 ? (int)p.a.prefix_len : 0;
    r.low = 0;
  } else {
    const int64_t cap = p.a.table_width * p.a.page_size;
    r.end = (int)max((int64_t)0, min((int64_t)x.pos0 + x.ntok, cap));
    r.low = p.a.window > 0 ? (int)min(max((int64_t)0, x.pos0 - p.a.window + 1), (int64_t)r.end) : 0;
  }
  const int sinks = (int)min(p.a.sinks, (int64_t)r.low);
  r.w0 = r.low / BN;
  r.ns = min((sinks + BN - 1) / BN, r.w0);
  r.n = max(1, r.ns + (r.end + BN - 1) / BN - r.w0);
  return r;
}
// blocks (from the first) that tile t of a pair needs
__device__ __forceinline__ int tile_blocks(const Params &p, const Pair &x, const Blocks &k, int t) {
  const int rows = min(x.ntok - t * p.P, p.P);
  if (rows <= 0) return 0;
  if (x.seq < 0) return x.seq == -1 ? k.n : 0;
  const int end = (int)max((int64_t)0, min((int64_t)x.pos0 + t * p.P + rows, (int64_t)k.end));
  return end == 0 ? 0 : k.ns + max(0, (end + BN - 1) / BN - k.w0);
}

// The list of pairs.  With a prefix alone (own = 0) it follows from the sizes:
// 2 P tokens each, all of the prefix's blocks; else k_paged_tile.cu writes it.
struct List {
  const Params &p;
  const int64_t *head;
  const Pair *pairs;
  __device__ __forceinline__ int size() const {
    const int per = 2 * p.P;
    return p.own ? (int)head[0] : (int)((p.a.tokens + per - 1) / per);
  }
  __device__ __forceinline__ Pair pair(int u) const {
    const int per = 2 * p.P;
    return p.own ? pairs[u] : Pair{-1, u * per, min(per, (int)p.a.tokens - u * per), 0};
  }
  // blocks (per key head) before pair u
  __device__ __forceinline__ int64_t before(int u) const {
    return p.own ? head[1 + u] : u * max((int64_t)1, (p.a.prefix_len + BN - 1) / BN);
  }
  // blocks of the longest of n pairs
  __device__ __forceinline__ int64_t longest(int n) const { return p.own ? head[2 + n] : before(1); }
};

// ---- segments: what a CTA's share holds of each unit -----------------------------
struct Segment {
  Pair x;
  Blocks k;
  int u, hk, k0, k1;  // pair, key head, blocks of it
  bool all;           // the whole unit
  int slot;           // of its partial
};
// The units' blocks are shared evenly over the CTAs, which cuts units: partials are
// written and joined, and a CTA may get many short units, each with its own start and
// end.  Or a CTA takes whole units, the last pairs first (under a causal mask the
// longest), the next when it has done one.  Cutting costs some 3 blocks' time, and 6
// for each unit that a CTA gets (up to 4); staying whole costs what the last units
// take beyond an equal share, half a unit where lengths vary.  The cheaper one, by
// that estimate.  Measured, us, cut and whole (32 / 8 heads of 128 bf16): 512 tokens
// 32 / 20, 1024 40 / 28, 2048 80 / 46, 2 x 2048 133 / 80, 8 x 128 after 4000 each 94 /
// 75; 128 after 2000 36 / 43, 512 after 4000 61 / 76, 8 x 160 after 4000 121 / 136.
constexpr int WHOLE = 6;  // units per CTA from which they always stay whole
__device__ __forceinline__ bool stay_whole(int64_t total, int64_t longest, int units, int ctas) {
  if (units >= WHOLE * ctas) return true;
  // in blocks times CTAs
  const int rounds = (units + ctas - 1) / ctas;
  const int64_t one = longest * ctas, whole = rounds == 1 ? one : min(rounds * one, total + one / 2);
  return whole <= total + 3 * ctas + 6 * min(units, 4 * ctas);
}
struct Walk {
  const Params &p;
  const List list;
  int pairs, c, units;
  Split split;
  int64_t f, f0, f1;
  bool whole;
  __device__ __forceinline__ Walk(const Params &q, int cta) : Walk(q, cta, q.head, q.pairs) {}
  __device__ __forceinline__ Walk(const Params &q, int cta, const int64_t *head, const Pair *items)
      : p(q), list{q, head, items}, pairs(list.size()), c(cta), units(pairs * (int)p.a.kv_heads),
        split(list.before(pairs) * p.a.kv_heads, p.max_ctas) {
    whole = stay_whole(split.total, list.longest(pairs), units, p.max_ctas);
    f0 = c < split.ctas ? split.first(c) : 0;
    f1 = c < split.ctas ? split.first(c + 1) : 0;
    f = f0;
  }
  __device__ __forceinline__ Parts parts(int u, int hk, int64_t n) const {
    const int unit = u * (int)p.a.kv_heads + hk;
    if (whole) return Parts{1, 0, 2 * p.max_ctas + unit};
    return parts_of(split, list.before(u) * p.a.kv_heads + hk * n, n, p.max_ctas, unit);
  }
  // unit that holds block `at`: a whole warp looks, 32 pivots at a time
  __device__ __forceinline__ void locate(int64_t at, Segment &s, int lane) const {
    const int64_t row = quotient(at, p.a.kv_heads);  // pairs are kv_heads * n blocks long
    int lo = 0, n = pairs;
    while (n > 1) {
      const int step = (n + 31) / 32, i = lane * step;
      const uint32_t m = __ballot_sync(0xffffffffu, i < n && list.before(lo + min(i, n - 1)) <= row);
      const int last = 31 - __clz(m | 1u);
      lo += last * step;
      n = min(step, n - last * step);
    }
    set(lo, s);
    const int in = (int)(at - list.before(lo) * p.a.kv_heads);
    s.hk = in / s.k.n;
    s.k0 = in - s.hk * s.k.n;
  }
  __device__ __forceinline__ void set(int u, Segment &s) const {
    s.u = u;
    s.x = list.pair(u);
    s.k = blocks_of(p, s.x);
  }
  // the next segment of the share (a whole warp)
  __device__ __forceinline__ bool next(Segment &s, int lane) {
    if (whole) {
      int i = c;
      if (!p.own || p.inside) {  // all of a length, or one each
        i += (int)(f - f0) * p.max_ctas;
      } else if (f != f0) {  // the next that no CTA has
        if (lane == 0) i = atomicAdd(p.next, 1);
        i = __shfl_sync(0xffffffffu, i, 0);
      }
      ++f;
      if (i >= units) return false;
      i = units - 1 - i;
      set(i / (int)p.a.kv_heads, s);
      s.hk = i % (int)p.a.kv_heads;
      s.k0 = 0;
      s.k1 = s.k.n;
      s.all = true;
      s.slot = 2 * p.max_ctas + i;
      return true;
    }
    if (f >= f1) return false;
    if (f == f0) {
      locate(f, s, lane);
    } else {  // a unit ended with the segment before
      s.k0 = 0;
      if (++s.hk == (int)p.a.kv_heads) {
        s.hk = 0;
        set(s.u + 1, s);
      }
    }
    s.k1 = (int)min((int64_t)s.k.n, s.k0 + (f1 - f));
    s.all = s.k0 == 0 && s.k1 == s.k.n;
    s.slot = s.all ? 2 * p.max_ctas + s.u * (int)p.a.kv_heads + s.hk : 2 * c + (f != f0);
    f += s.k1 - s.k0;
    return true;
  }
};

// floats of one partial: the rows of both tiles, then their (max, sum)
constexpr int slot_floats(int dp) { return 2 * BM * (dp + 2); }

}  // namespace several

bool tile_form(const Args &a);     // by the sizes
bool tile_strides(const Args &a);  // whether TMA can describe the operands
// `own`: the sequences' own keys, `prefix`: the shared prefix's; `keep`: every
// result stays a partial in the workspace
size_t tile_workspace(const Args &a, int device, bool own, bool prefix, bool keep);
int tile_params(const Args &a, int device, void *workspace, bool own, bool prefix, bool keep, several::Params *p);
int tile_launch(const several::Params &p, cudaStream_t st, int device);

// a shared prefix (k_paged_prefix.cu)
size_t prefix_workspace(const Args &a, int device);
int prefix_run(const Args &a, cudaStream_t st, int device);
int tile_read_and_clear_error(int *flag);

}  // namespace pattn
}  // namespace nkb
