// Paged attention of several tokens per sequence on the 5th-generation tensor
// cores (bf16, fp16, head dimensions up to 128):
//   out[t, h] = sum_j softmax_j(q[t, h] . k_j * scale) v_j
// over the keys j that token t sees through the page table (causal, with an
// optional window and first tokens), online softmax with fp32 statistics.
//
// The G query heads of a key head and P = 128 / G consecutive tokens are the
// rows of one 128-row tile, so every key row that is fetched serves all of
// them; a CTA works on two tiles (a "pair" of 2 P tokens) against blocks of 128
// keys.  The blocks of all (pair, key head) units form one run that the
// resident CTAs split evenly, whatever the lengths; a unit that crosses a
// share's end is joined from partials by a second kernel.  Lengths are read on
// the device, where the pairs are listed: by a small kernel, a short list by each CTA.
//
// A block is taken in two halves of 64 keys, each with its own score buffer, so
// that the scores of the next half are there when a softmax ends: the softmax
// warps wait for no product of their own half.  Warps of a CTA:
//   8      walks the CTA's share, hands its segments to the others through a small
//          ring, and produces: TMA loads of Q (both tiles) and, page by page, of
//          K and V into rings of stages that are released separately;
//   9, 10  issue the products of tile A and of tile B: S(0)
//          S(1), then per half PV(h) S(h + 2); warp 9 owns the TMEM;
//   11     sees to V: rows that no token of the pair sees become zeros;
//   0-3, 4-7  softmax of tile A and of tile B, one thread per row: scores from
//          TMEM, mask, running maximum (raised only when it grows by more than
//          2^8, O is then scaled in TMEM), exp2, P as 16-bit pairs over the
//          scores; at a segment's end O / l to memory, or the partial.
// Keys that no row of the CTA sees may hold anything (another sequence's rows,
// infinities, NaN): their scores are replaced; pages of which no key is seen are
// not read (TMA fills zeros), and the unseen V rows of the others are set to
// zero in shared memory before the product that would multiply them by zero.
// TMEM: two score buffers of 64 columns and O of up to 128 for each tile.  Every wait is bounded.
//
// What bounds it is the softmax between the two products: the exponentials take as
// many cycles as the products at head dimension 128 and twice as many at 64, so
// 3/8 of them are polynomials on the FMA pipe.  Measured (replays of a graph of 30
// calls, then one call after another on changing inputs): 4 prompts of 2048 tokens,
// window 1024, 32 / 8 heads of 128 bf16, 135 and 154 us, 766 and 671 TFLOP/s of the
// keys seen (tensor pipe busy 41 %, issue slots 41 %); 500 tokens over 16400 keys,
// 32 / 4 heads of 64 fp16, 129 and 132 us with 15 of them in the join, 511 and 500
// TFLOP/s (tensor 25 %, issue 44 %).
#include <math_constants.h>

#include "paged_attn.cuh"
#include "sm100.cuh"

namespace nkb {
namespace pattn {
namespace {

using namespace sm100;

using namespace several;

constexpr int BH = 64;  // keys of a half
constexpr int W_PROD = 8, W_MMA = 9, W_FIX = 11, THREADS = 384;
constexpr int RING = 4;  // segments
constexpr int HALF = 128 * 64 * 2;  // 128 rows x 64 columns, 128-byte swizzle
constexpr uint32_t T_S = 0, T_O = 256, TMEM_COLS = 512;
constexpr float RESCALE = 8.f;  // log2 headroom before the running maximum is raised

__device__ int g_tile_error = 0;

// A short list is made by each CTA of the tile kernel for itself, in its shared
// memory: that takes a microsecond or two, the kernel above and its launch four.
constexpr int LIST = 256;  // pairs, and sequences
struct OwnList {
  int64_t head[LIST + 3];
  Pair pairs[LIST];
  int seq_pairs[LIST + 2];
};

template <int DP>
struct Cfg {
  static constexpr int HALVES = DP / 64, TILE = HALVES * HALF, STAGES = DP == 128 ? 2 : 4;
  static constexpr int OFF_K = 2 * TILE, OFF_V = OFF_K + STAGES * TILE, OFF_BAR = OFF_V + STAGES * TILE;
  static constexpr int OFF_ITEMS = OFF_BAR + 448;
  static constexpr int OFF_LIST = OFF_ITEMS + RING * 64;
  static constexpr int SMEM = 1024 + OFF_LIST + (int)sizeof(OwnList);
  static constexpr int SLOT = slot_floats(DP);
};

// ---- the list of pairs ---------------------------------------------------------
constexpr int SCHED = 1024;

// exclusive sum over the block; *total gets the sum
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *total) {
  __shared__ int64_t s[SCHED / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, w);
    if (lane >= w) x += y;
  }
  __syncthreads();
  if (lane == 31) s[warp] = x;
  __syncthreads();
  int64_t y = s[lane];  // the warps' sums, scanned by every warp
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const int64_t z = __shfl_up_sync(0xffffffffu, y, w);
    if (lane >= w) y += z;
  }
  *total = __shfl_sync(0xffffffffu, y, 31);
  const int64_t before = __shfl_sync(0xffffffffu, y, max(warp - 1, 0));
  return (warp ? before : 0) + x - v;
}

// tokens of list entry i: those before the sequences, sequence i - 1, those after
__device__ __forceinline__ void tokens_of(const Args &a, int i, int &first, int &n) {
  const int B = (int)a.seqs, T = (int)a.tokens;
  const int lo = i == 0 ? 0 : a.q_start[i - 1], hi = i > B ? T : a.q_start[i];
  first = max(0, min(lo, T));
  n = max(0, min(hi, T) - first);
}

// Who lists: a block of SCHED threads, or one warp.
struct Block {
  static constexpr int N = SCHED;
  static __device__ __forceinline__ int id() { return threadIdx.x; }
  static __device__ __forceinline__ int64_t scan(int64_t v, int64_t *total) { return block_scan(v, total); }
  static __device__ __forceinline__ int largest(int v) {
    __shared__ int s;
    if (threadIdx.x == 0) s = 0;
    __syncthreads();
    atomicMax(&s, v);
    __syncthreads();
    return s;
  }
  static __device__ __forceinline__ void sync() { __syncthreads(); }
};
struct Warp {
  static constexpr int N = 32;
  static __device__ __forceinline__ int id() { return threadIdx.x & 31; }
  static __device__ __forceinline__ int64_t scan(int64_t v, int64_t *total) {
    int64_t x = v;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, w);
      if (id() >= w) x += y;
    }
    *total = __shfl_sync(0xffffffffu, x, 31);
    return x - v;
  }
  static __device__ __forceinline__ int largest(int v) { return __reduce_max_sync(0xffffffffu, v); }
  static __device__ __forceinline__ void sync() { __syncwarp(); }
};
template <class Group>
__device__ __forceinline__ void list_pairs(const Params &p, int64_t *head, Pair *pairs, int *seq_pairs) {
  const Args &a = p.a;
  const int per = 2 * p.P, B = (int)a.seqs, T = (int)a.tokens;
  const int lists = B + 2, front = p.prefix ? (T + per - 1) / per : 0;
  int64_t npairs = front;
  for (int base = 0; base < lists; base += Group::N) {
    const int i = base + Group::id();
    int first, n = 0;
    if (i < lists) tokens_of(a, i, first, n);
    int64_t all;
    const int64_t at = npairs + Group::scan((n + per - 1) / per, &all);
    if (i < lists) seq_pairs[i] = (int)min(at, (int64_t)p.max_pairs);
    npairs += all;
  }
  // the list holds max_pairs: q_start entries that overlap, which no caller means, would need more
  const int U = (int)min(npairs, (int64_t)p.max_pairs);
  Group::sync();
  int64_t blocks = 0;
  int longest = 0;
  for (int base = 0; base < U; base += Group::N) {
    const int u = base + Group::id();
    int64_t nb = 0;
    Pair x = {-2, 0, 0, 0};
    if (u < front) {
      x = {-1, u * per, min(per, T - u * per), 0};
    } else if (u < U) {
      int lo = 0, hi = lists - 1;  // the last list that begins at or before u
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (seq_pairs[mid] <= u) lo = mid;
        else hi = mid - 1;
      }
      int first, n;
      tokens_of(a, lo, first, n);
      const int off = (u - seq_pairs[lo]) * per;
      x.tok0 = first + off;
      x.ntok = max(0, min(per, n - off));
      if (lo >= 1 && lo <= B) {
        x.seq = lo - 1;
        x.pos0 = a.kv_len[lo - 1] - n + off;
      }
    }
    if (u < U) {
      nb = blocks_of(p, x).n;
      longest = max(longest, (int)nb);
      pairs[u] = x;
    }
    int64_t all;
    const int64_t at = blocks + Group::scan(nb, &all);
    if (u < U) head[1 + u] = at;
    blocks += all;
  }
  longest = Group::largest(longest);
  if (Group::id() == 0) {
    head[0] = U;
    head[1 + U] = blocks;
    head[2 + U] = longest;
  }
  Group::sync();
}

__global__ void __launch_bounds__(SCHED) pairs_kernel(const __grid_constant__ Params p) {
  pdl_trigger();
  list_pairs<Block>(p, p.head, p.pairs, p.seq_pairs);
  if (threadIdx.x == 0) *p.next = p.max_ctas;  // the CTAs' first units are their own numbers
}

__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
  return mbar_wait(bar, parity, abort_flag, &g_tile_error);
}
__device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
  return __all_sync(0xffffffffu, wait(bar, parity, abort_flag));
}
// instruction descriptor, kind::f16, fp32 accumulator: both operands bf16 or both fp16
template <class T>
__device__ __forceinline__ constexpr uint32_t idesc(int M, int N, int b_mn_major) {
  constexpr uint32_t fmt = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

// Products and commits of a whole warp, issued by its elected lane: the warp
// stays converged and the descriptors warp-uniform, so that no operand has to be
// moved out of a diverged thread's registers (in an `if (lane == 0)` an issue
// took about 100 cycles, which bounded the kernel).
__device__ __forceinline__ void warp_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void warp_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void warp_commit(uint64_t *bar) {
  asm volatile(
      "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar))
      : "memory");
}

// A segment as the roles need it.
struct Item {
  int seq, tok0, ntok, pos0, hk;
  int end, low, ns, w0;  // Blocks
  int k0, n;             // first block, number of blocks; n = 0: the share is done
  int nb_a, nb_b;        // blocks that each tile needs
  int final, slot;
};

// Two fp32 values as one operand of the packed instructions.
__device__ __forceinline__ uint64_t pair2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair2(uint64_t v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// the largest of three, NaN if one is NaN
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^y for two values on the FMA pipe: y = n + r with |r| <= 1/2, 2^r by its
// minimax polynomial (least squares reweighted to an even relative error: 7.5e-5
// for degree 3, 2.7e-6 for degree 4, a tenth of the rounding of P to bf16 and to
// fp16), n added to the exponent.  y below -126 gives 2^-126.  P is rounded because the
// matrix product takes both operands in one type; the sums keep fp32 terms.  Outputs
// are 0.0021 (bf16) and 0.00029 (fp16) from 64-bit values in the root mean square, where
// fp32 probabilities and exact exponentials give 0.0016 and 0.00021.
template <class T>
__device__ __forceinline__ void exp2_poly(uint64_t y2, float &e0, float &e1) {
  constexpr bool fine = std::is_same<T, __half>::value;
  float y0, y1, t0, t1;
  unpair2(y2, y0, y1);
  y2 = pair2(fmaxf(y0, -126.f), fmaxf(y1, -126.f));
  const uint64_t t2 = add2(y2, pair2(12582912.f, 12582912.f));           // 1.5 * 2^23: n in the low bits
  const uint64_t r2 = fma2(add2(t2, pair2(-12582912.f, -12582912.f)), pair2(-1.f, -1.f), y2);
  auto c = [](float x) { return pair2(x, x); };
  uint64_t q;
  if (fine) {
    q = fma2(c(9.570101276040077e-3f), r2, c(5.591786280274391e-2f));
    q = fma2(q, r2, c(0.240247443318367f));
    q = fma2(q, r2, c(0.6931217908859253f));
    q = fma2(q, r2, c(0.9999992847442627f));
  } else {
    q = fma2(c(5.51716610789299e-2f), r2, c(0.2426111400127411f));
    q = fma2(q, r2, c(0.6932609677314758f));
    q = fma2(q, r2, c(0.9999280571937561f));
  }
  unpair2(t2, t0, t1);
  unpair2(q, e0, e1);
  e0 = __int_as_float(__float_as_int(e0) + (__float_as_int(t0) << 23));
  e1 = __int_as_float(__float_as_int(e1) + (__float_as_int(t1) << 23));
}

// 32 bytes of one row (a whole sector), or two halves where they are only
// aligned to 16
__device__ __forceinline__ void store32(void *p, const uint32_t *v, bool wide) {
  if (wide)
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  else {
    static_cast<uint4 *>(p)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    static_cast<uint4 *>(p)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

// Descriptors whose address part moves by a constant.
struct Desc {
  uint32_t lo, hi;
  __device__ __forceinline__ explicit Desc(uint64_t d) : lo((uint32_t)d), hi((uint32_t)(d >> 32)) {}
  __device__ __forceinline__ uint64_t at(uint32_t bytes) const {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo + (bytes >> 4)), "r"(hi));
    return r;
  }
};

// INSIDE: the CTA lists the pairs for itself.  (Two kernels, not a branch: with the
// listing beside it the others' walk took 1 to 4 us more per call.)
template <class T, int DP, bool INSIDE>
__global__ void __launch_bounds__(THREADS, 1)
    tile_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                const __grid_constant__ CUtensorMap mv, const __grid_constant__ Params p) {
  using C = Cfg<DP>;
  constexpr int ST = C::STAGES;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::OFF_BAR);
  // [tile][score buffer] where a tile has two
  uint64_t *q_full = bars, *q_empty = bars + 1, *s_full = bars + 2, *p_ready = bars + 6, *o_done = bars + 10,
           *o_free = bars + 14, *i_full = bars + 16, *i_empty = i_full + RING, *k_full = i_empty + RING,
           *k_empty = k_full + ST, *v_full = k_empty + ST, *v_empty = v_full + ST, *v_ready = v_empty + ST,
           *b_go = v_ready + ST;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(b_go + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  Item *ring = reinterpret_cast<Item *>(smem + C::OFF_ITEMS);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const Args &a = p.a;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);  // both issuers
    mbar_init(b_go, 1);
    for (int t = 0; t < 2; ++t) {
      for (int j = 0; j < 2; ++j) {
        mbar_init(&s_full[2 * t + j], 1);
        mbar_init(&p_ready[2 * t + j], BM);
        mbar_init(&o_done[2 * t + j], 1);
      }
      mbar_init(&o_free[t], BM);
    }
    for (int s = 0; s < RING; ++s) {
      mbar_init(&i_full[s], 1);
      mbar_init(&i_empty[s], 11);  // two issuers, V's warp, eight softmax warps
    }
    for (int s = 0; s < ST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 2);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 2);
      mbar_init(&v_ready[s], 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == W_PROD && lane == 0) {
    prefetch_map(&mq);
    prefetch_map(&mk);
    prefetch_map(&mv);
  }
  if (warp == W_MMA) tmem_alloc(tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();
  bool ok = true;
  uint32_t items = 0;  // segments taken so far
  // the next segment, from the ring (a whole warp)
  auto take = [&](Item &x) {
    const int i = items % RING;
    if (!(ok = wait_warp(&i_full[i], (items / RING) & 1, abort_flag))) return false;
    x = ring[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(&i_empty[i]);
    ++items;
    return x.n > 0;
  };
  auto block_of = [](const Item &x, int i) { return i < x.ns ? i : x.w0 + i - x.ns; };

  if (warp >= W_PROD) {
    if (warp == W_PROD) {
      // ---------------- segments of this CTA's share, TMA producer ----------------
      const int ps = (int)a.page_size, box = min(ps, BN), npb = BN / box;  // pages (or page parts) per block
      uint32_t segs = 0, blk = 0;
      const int64_t *head = p.head;
      const Pair *pairs = p.pairs;
      if constexpr (INSIDE) {
        OwnList *own = reinterpret_cast<OwnList *>(smem + C::OFF_LIST);
        list_pairs<Warp>(p, own->head, own->pairs, own->seq_pairs);
        if (blockIdx.x == 0) {  // for the join
          for (int i = lane; i < own->head[0] + 3; i += 32) p.head[i] = own->head[i];
          for (int i = lane; i < own->head[0]; i += 32) p.pairs[i] = own->pairs[i];
        }
        head = own->head;
        pairs = own->pairs;
      }
      Walk walk(p, blockIdx.x, head, pairs);
      Segment s;
      while (ok) {
        const bool more = walk.next(s, lane);
        const int slot_i = items % RING;
        if (!(ok = wait_warp(&i_empty[slot_i], ((items / RING) & 1) ^ 1, abort_flag))) break;
        Item x = {};
        if (more) {
          x = {s.x.seq, s.x.tok0, s.x.ntok, s.x.pos0, s.hk, s.k.end, s.k.low, s.k.ns, s.k.w0, s.k0, s.k1 - s.k0, 0, 0,
               s.all && !p.keep, s.slot};
          x.nb_a = max(0, min(x.n, tile_blocks(p, s.x, s.k, 0) - s.k0));
          x.nb_b = max(0, min(x.n, tile_blocks(p, s.x, s.k, 1) - s.k0));
        }
        if (lane == 0) {
          ring[slot_i] = x;
          mbar_arrive(&i_full[slot_i]);
        }
        __syncwarp();
        ++items;
        if (!more) break;
        const int32_t *table = x.seq < 0 ? a.prefix_pages : a.page_table + x.seq * a.table_stride;
        const int sinks = (int)min(a.sinks, (int64_t)x.end);
        // page of this lane's part of block i; one past the cache (zeros) where no key of it is seen
        auto page_of = [&](int i) {
          const int64_t key = (int64_t)block_of(x, i) * BN + lane * box;
          int id = -1;
          if (i < x.k0 + x.n && lane < npb && key < x.end && (key + box > x.low || key < sinks)) id = table[key >> p.page_shift];
          return paged::page_ok(id, a.pages) ? id : (int)a.pages;
        };
        int next = page_of(x.k0);
        if (!(ok = wait_warp(q_empty, (segs & 1) ^ 1, abort_flag))) break;
        if (lane == 0) {
          const int tiles = x.ntok > p.P ? 2 : 1;
          mbar_expect_tx(q_full, tiles * C::HALVES * 128 * p.G * p.P);
          for (int t = 0; t < tiles; ++t)
            for (int j = 0; j < C::HALVES; ++j)
              tma_load_4d(smem + t * C::TILE + j * HALF, &mq, q_full, j * 64, 0, x.hk, x.tok0 + t * p.P);
        }
        ++segs;
        for (int i = x.k0; i < x.k0 + x.n; ++i, ++blk) {
          const int st = blk % ST, page = next;
          const uint32_t par = ((blk / ST) & 1) ^ 1;
          const int slot = (block_of(x, i) * BN + lane * box) & (ps - 1);
          next = page_of(i + 1);
          uint8_t *kt = smem + C::OFF_K + st * C::TILE + lane * box * 128, *vt = smem + C::OFF_V + st * C::TILE + lane * box * 128;
          if (!(ok = wait_warp(&k_empty[st], par, abort_flag))) break;
          if (lane == 0) mbar_expect_tx(&k_full[st], C::TILE);
          __syncwarp();
          if (lane < npb)
            for (int j = 0; j < C::HALVES; ++j) tma_load_4d(kt + j * HALF, &mk, &k_full[st], j * 64, slot, x.hk, page);
          if (!(ok = wait_warp(&v_empty[st], par, abort_flag))) break;
          if (lane == 0) mbar_expect_tx(&v_full[st], C::TILE);
          __syncwarp();
          if (lane < npb)
            for (int j = 0; j < C::HALVES; ++j) tma_load_4d(vt + j * HALF, &mv, &v_full[st], j * 64, slot, x.hk, page);
        }
      }
    } else if (warp == W_FIX) {
      // ---------------- V rows that no token of the pair sees ----------------
      uint32_t blk = 0;
      Item x;
      while (ok && take(x)) {
        const int sinks = (int)min(a.sinks, (int64_t)x.end);
        for (int i = x.k0; i < x.k0 + x.n; ++i, ++blk) {
          const int st = blk % ST, key0 = block_of(x, i) * BN;
          if (!(ok = wait_warp(&v_full[st], (blk / ST) & 1, abort_flag))) break;
          if (key0 + BN > x.end || (key0 < x.low && key0 + BN > sinks)) {
            // four rows at a time, eight lanes on the 128 bytes of a row
            for (int r = lane / 8; r < BN; r += 4) {
              const int key = key0 + r;
              if (key < x.end && (key >= x.low || key < sinks)) continue;
              uint8_t *row = smem + C::OFF_V + st * C::TILE + r * 128 + lane % 8 * 16;
#pragma unroll
              for (int j = 0; j < C::HALVES; ++j) *reinterpret_cast<uint4 *>(row + j * HALF) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (lane == 0) mbar_arrive(&v_ready[st]);
        }
      }
    } else {
      // ---------------- MMA issuer of tile t ----------------
      constexpr uint32_t ID_S = idesc<T>(128, BH, 0), ID_O = idesc<T>(128, DP, 1);
      const int t = __shfl_sync(0xffffffffu, warp, 0) - W_MMA;
      const Desc dq(smem_desc(smem_u32(smem + t * C::TILE), 16, 1024)), dk(smem_desc(smem_u32(smem + C::OFF_K), 16, 1024)),
          dv(smem_desc(smem_u32(smem + C::OFF_V), HALF, 1024));
      const uint32_t ts = tmem + T_S + t * 128, to = tmem + T_O + t * 128;
      uint32_t segs = 0, blk = 0, cnt = 0, outs = 0, turns = 0;
      Item x;
      while (ok && take(x)) {
        const int n = __shfl_sync(0xffffffffu, x.n, 0), nb = __shfl_sync(0xffffffffu, t ? x.nb_b : x.nb_a, 0);
        const bool paired = __shfl_sync(0xffffffffu, x.nb_a > 0 && x.nb_b > 0, 0);
        // tile B begins when the softmax of A has done its first half: in step, both would want the special-function
        // units at one time and the tensor cores at another.  Only where both tiles have a block: A's arrival is then
        // behind this segment's Q, which is loaded when B has released the Q before, past its last wait here.  Without
        // a block A would arrive as soon as it has the segment, and twice before B looks: a parity that is the old one.
        if (paired && t == 1 && !(ok = wait_warp(b_go, turns++ & 1, abort_flag))) break;
        auto stage = [&](int c) { return (blk + c) % ST; };
        auto full = [&](uint64_t *bar, int c) { return wait_warp(&bar[stage(c)], ((blk + c) / ST) & 1, abort_flag); };
        auto qk = [&](int c, int j) {  // S = Q K^T of half j of block c
          const Desc k(dk.at(stage(c) * C::TILE + j * BH * 128));
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk) {
            const uint32_t off = (kk >> 2) * HALF + (kk & 3) * 32;
            warp_mma(ts + j * BH, dq.at(off), k.at(off), ID_S, kk > 0);
          }
          warp_commit(&s_full[2 * t + j]);
        };
        auto pv = [&](int c, int j) {  // O += P V
          const Desc v(dv.at(stage(c) * C::TILE + j * BH * 128));
#pragma unroll
          for (int kk = 0; kk < BH / 16; ++kk)
            warp_mma_ts(to, ts + j * BH + kk * 8, v.at(kk * 2048), ID_O, (c > 0 || j > 0 || kk > 0) ? 1u : 0u);
          warp_commit(&o_done[2 * t + j]);
        };
        if (!(ok = wait_warp(q_full, segs & 1, abort_flag) && full(k_full, 0))) break;
        ++segs;
        tc_fence_after();
        if (nb > 0) {
          qk(0, 0);
          qk(0, 1);
        }
        warp_commit(&k_empty[stage(0)]);
        if (n == 1) warp_commit(q_empty);
        for (int c = 0; c < n; ++c) {
          // a block that this tile does not need is waited for all the same: its stages are released in order
          if (!(ok = full(v_ready, c))) break;
          if (c < nb) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // P of the half is written; before a segment's first product, O of the segment before is read
              if (!(ok = wait_warp(&p_ready[2 * t + j], cnt & 1, abort_flag) &&
                         (c > 0 || j > 0 || outs == 0 || wait_warp(&o_free[t], (outs - 1) & 1, abort_flag))))
                break;
              tc_fence_after();
              pv(c, j);
              if (c + 1 < nb) {
                if (j == 0 && !(ok = full(k_full, c + 1))) break;
                tc_fence_after();
                qk(c + 1, j);
              }
            }
            if (!ok) break;
            ++cnt;
          }
          warp_commit(&v_empty[stage(c)]);
          if (c + 1 < n) {
            if (c + 1 >= nb && !(ok = full(k_full, c + 1))) break;
            warp_commit(&k_empty[stage(c + 1)]);
            if (c + 2 == n) warp_commit(q_empty);
          }
        }
        blk += n;
        outs += nb > 0;
      }
    }
  } else {
    // ---------------- softmax and results: tile t, row r ----------------
    const int t = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t rows = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t s_col = rows + T_S + t * 128, o_col = rows + T_O + t * 128;
    const int g = r % p.G, tok = t * p.P + r / p.G;  // query head in the group, token in the pair
    const uint64_t scale2 = pair2(p.scale_log2, p.scale_log2);
    uint32_t blk = 0, cnt = 0;
    Item x;
    while (ok && take(x)) {
      const int nb = t ? x.nb_b : x.nb_a;
      const bool row_ok = r < p.P * p.G && tok < x.ntok;
      // keys that the row sees: [lo, hi), and below `first`
      int hi = 0, lo = 0, first = 0;
      if (row_ok) {
        const int64_t pos = (int64_t)x.pos0 + tok;
        hi = x.seq < 0 ? x.end : (int)max((int64_t)0, min(pos + 1, (int64_t)x.end));
        if (x.seq >= 0 && a.window > 0) {
          lo = (int)min(max((int64_t)0, pos - a.window + 1), (int64_t)hi);
          first = (int)min(a.sinks, (int64_t)hi);
        }
      }
      // halves that need no mask: from the last row's first key to the first row's last one
      const int plain_lo = __reduce_max_sync(0xffffffffu, lo), plain_hi = __reduce_min_sync(0xffffffffu, hi);
      float m = -INFINITY, l = 0.f;  // running (possibly stale) maximum in log2 units, and sum
      for (int h = 0; h < 2 * nb; ++h, ++cnt) {
        const int c = h >> 1, j = h & 1, key0 = block_of(x, x.k0 + c) * BN + j * BH;
        const uint32_t sc = s_col + j * BH;
        // the scores, and the product of the half before last: every phase of o_done is waited for in turn, so
        // that the parity of a later wait (below) cannot be that of an older phase
        ok = wait(&s_full[2 * t + j], (cnt >> 1) & 1, abort_flag) &&
             (h < 2 || wait(&o_done[2 * t + j], ((cnt >> 1) - 1) & 1, abort_flag));
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc_fence_after();
        uint32_t v[BH];
        tmem_ld32_nw(sc, v);
        tmem_ld32_nw(sc + 32, v + 32);
        tmem_ld_wait();
        const bool masked = key0 < plain_lo || key0 + BH > plain_hi;
        if (masked) {
          // a bit per key: below hi, and from lo or below first
          const int hk = hi - key0, w = lo - key0, f = first - key0;
          auto below = [](int n) -> uint32_t { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t bits = below(hk - 32 * i) & (~below(w - 32 * i) | below(f - 32 * i));
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(bits >> e & 1)) v[32 * i + e] = 0xff800000u;
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < BH; e += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mx4[i] = max3(mx4[i], __uint_as_float(v[e + 2 * i]), __uint_as_float(v[e + 2 * i + 1]));
        const float mx = max3(max3(mx4[0], mx4[1], mx4[2]), mx4[3], -INFINITY) * p.scale_log2;
        const bool raise = !(mx <= m + RESCALE);
        bool exact = masked;  // zeros have to be zeros: masked scores, and rows whose scores are all -inf
        if (__any_sync(0xffffffffu, raise || (!masked && mx == -INFINITY))) {
          // a score of NaN or +inf makes the maximum NaN, and so all of the row: the polynomials would take it for 2^-126
          const float m_new = raise ? (mx == INFINITY ? CUDART_NAN_F : mx) : m;
          const float alpha = m == -INFINITY ? 0.f : raise ? ex2(m - m_new) : 1.f;
          // (rows that have seen no key so far have O = 0 already)
          if (h > 0 && __any_sync(0xffffffffu, raise && m > -INFINITY)) {
            if (!(ok = wait_warp(&o_done[2 * t + (j ^ 1)], ((cnt - 1) >> 1) & 1, abort_flag))) break;
            tc_fence_after();
#pragma unroll 1
            for (int i = 0; i < DP / 16; ++i) {
              uint32_t o[16];
              tmem_ld16(o_col + i * 16, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st16(o_col + i * 16, o);
            }
            tmem_st_wait();
          }
          l *= alpha;
          m = m_new;
          exact |= __any_sync(0xffffffffu, m == -INFINITY) != 0;
        }
        const float mm = base_of(m);
        const uint64_t base2 = pair2(-mm, -mm);
        uint64_t l2[2] = {0, 0};
        // of every eight pairs, `POLY` on the FMA pipe: the special-function unit alone would take 64 x 8 cycles a warp
        auto exps = [&](auto poly) {
#pragma unroll
          for (int e = 0; e < BH; e += 2) {
            float e0, e1;
            const uint64_t y2 = fma2(pair2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), scale2, base2);
            if (decltype(poly)::value && ((e >> 1) & 7) % 3 == 1) {
              exp2_poly<T>(y2, e0, e1);
            } else {
              unpair2(y2, e0, e1);
              e0 = ex2(e0);
              e1 = ex2(e1);
            }
            l2[(e >> 1) & 1] = add2(l2[(e >> 1) & 1], pair2(e0, e1));
            v[e / 2] = pack<T>(e0, e1);
          }
        };
        if (exact) exps(std::false_type{});
        else exps(std::true_type{});
        tmem_st16(sc, v);
        tmem_st16(sc + 16, v + 16);
        float s0, s1, s2, s3;
        unpair2(l2[0], s0, s1);
        unpair2(l2[1], s2, s3);
        l += (s0 + s1) + (s2 + s3);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_ready[2 * t + j]);
        if (h == 0 && warp == 0 && lane == 0 && x.nb_b > 0) mbar_arrive(b_go);
      }
      if (!ok) break;
      blk += x.n;
      if (nb > 0) {
        const uint32_t last = ((cnt >> 1) - 1) & 1;
        if (!(ok = wait_warp(&o_done[2 * t], last, abort_flag) && wait_warp(&o_done[2 * t + 1], last, abort_flag))) break;
        tc_fence_after();
      }
      uint32_t o[DP];
#pragma unroll
      for (int i = 0; i < DP; ++i) o[i] = 0;
      if (nb > 0) {
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) tmem_ld32_nw(o_col + i * 32, o + i * 32);
        tmem_ld_wait();
        tc_fence_before();
        mbar_arrive(&o_free[t]);  // the next segment's products may go on
      }
      if (!row_ok) continue;
      if (l == 0.f) {  // saw nothing: zeros, where its zero weights have met an infinity or NaN that others see
#pragma unroll
        for (int i = 0; i < DP; ++i) o[i] = 0;
      }
      const int D = (int)a.head_dim;
      if (x.final) {
        const float inv = inverse(l);
        T *dst = static_cast<T *>(a.out) + (x.tok0 + tok) * a.out_token + (x.hk * p.G + g) * a.out_head;
#pragma unroll
        for (int i = 0; i < DP; i += 16) {
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            w[e] = pack<T>(__uint_as_float(o[i + 2 * e]) * inv, __uint_as_float(o[i + 2 * e + 1]) * inv);
          if (i + 16 <= D) store32(dst + i, w, p.wide);
          else if (i < D) *reinterpret_cast<uint4 *>(dst + i) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else {
        float *part = p.ws + (int64_t)x.slot * C::SLOT;
#pragma unroll
        for (int i = 0; i < DP; i += 8) store32(part + (t * BM + r) * DP + i, o + i, true);
        *reinterpret_cast<float2 *>(part + 2 * BM * DP + 2 * (t * BM + r)) = make_float2(m, l);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag && warp == W_PROD && lane == 0) {  // copies in flight land before the memory is given up
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000) {
    }
  }
  __syncthreads();
  if (warp == W_MMA) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// Joins the partials of the units that a share's end cuts: an item (c, y) is the
// unit cut by the beginning of CTA c's share, if that is the unit's first cut,
// and 32 of its rows.
constexpr int JOIN = 256;
template <class T, int DP>
__global__ void __launch_bounds__(JOIN) tile_join_kernel(const __grid_constant__ Params p) {
  using C = Cfg<DP>;
  constexpr int PARTS = 2 * BM / 32;
  pdl_wait();
  const Args &a = p.a;
  const Walk walk(p, 0);
  if (walk.whole) return;
  for (int item = blockIdx.x; item < (walk.split.ctas - 1) * PARTS; item += gridDim.x) {
    const int c = item / PARTS + 1;
    const int64_t cut = walk.split.first(c);
    Segment s;
    walk.locate(cut, s, threadIdx.x % 32);
    if (s.k0 == 0) continue;  // the share begins with the unit
    const Parts parts = parts_of(walk.split, cut - s.k0, s.k.n, p.max_ctas, 0);
    if (parts.c0 != c - 1) continue;
    for (int i = threadIdx.x; i < 32 * (DP / 4); i += JOIN) {
      const int row = item % PARTS * 32 + i / (DP / 4), d = i % (DP / 4) * 4, t = row / BM, r = row % BM;
      const int g = r % p.G, tok = t * p.P + r / p.G;
      if (r >= p.P * p.G || tok >= s.x.ntok || d >= (int)a.head_dim) continue;
      Joined<4> x;
      x.add(parts.n, [&](int j) {
        const float *slot = p.ws + (int64_t)parts.slot(j) * C::SLOT;
        return Partial{slot + row * DP + d, slot + 2 * BM * DP + 2 * row};
      });
      x.store(static_cast<T *>(a.out) + (s.x.tok0 + tok) * a.out_token + (s.hk * p.G + g) * a.out_head + d);
    }
  }
}

int log2_of(int64_t x) {
  int s = 0;
  while ((int64_t(1) << s) < x) ++s;
  return (int64_t(1) << s) == x ? s : -1;
}

// workspace: head | pairs | seq_pairs | partial slots, from its first 32-byte boundary
// (the partials are written 32 bytes at a time; a caller's alignment is 16)
constexpr size_t WS_ALIGN = 32, WS_SLACK = WS_ALIGN - 16;
struct Layout {
  size_t next, pairs, seqs, ws, bytes;
  int max_pairs;
};
Layout layout(const Args &a, int max_ctas, bool own, bool prefix, bool keep) {
  const int64_t per = 2 * (BM / (a.q_heads / a.kv_heads)), T = a.tokens;
  Layout x;
  // every sequence, and the tokens before and after them, may end in a part of a pair
  x.max_pairs = (int)((prefix ? (T + per - 1) / per : 0) + (own ? T / per + a.seqs + 2 : 0));
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  x.next = ((size_t)x.max_pairs + 3) * 8;
  x.pairs = up(x.next + 8);
  x.seqs = x.pairs + up((size_t)x.max_pairs * sizeof(Pair));
  x.ws = x.seqs + up((size_t)(own ? a.seqs + 2 : 0) * 4);
  const size_t slot = (a.head_dim <= 64 ? Cfg<64>::SLOT : Cfg<128>::SLOT) * sizeof(float);
  x.bytes = x.ws + (2 * (size_t)max_ctas + (keep ? (size_t)x.max_pairs * a.kv_heads : 0)) * slot + WS_SLACK;
  return x;
}

// (d, slot, head, page) map of a cache; unit dimensions get a valid stride
int cache_map(CUtensorMap *m, const void *ptr, const Args &a, int64_t page, int64_t slot, int64_t head) {
  const int64_t d8 = (a.head_dim + 7) / 8 * 8;
  const uint64_t dims[4] = {(uint64_t)a.head_dim, (uint64_t)a.page_size, (uint64_t)a.kv_heads, (uint64_t)a.pages};
  const uint64_t strides[3] = {(uint64_t)(a.page_size > 1 ? slot : d8), (uint64_t)(a.kv_heads > 1 ? head : d8),
                               (uint64_t)(a.pages > 1 ? page : d8)};
  const uint32_t box[4] = {64, (uint32_t)(a.page_size < BN ? a.page_size : BN), 1, 1};
  return make_bf16_map(m, ptr, 4, dims, strides, box);  // 16-bit elements, moved as they are
}

template <class T, int DP>
int launch(const Params &p, cudaStream_t st, int device) {
  static ContextOnce attr;
  if (int s = attr.run(device, []() -> int {
        NKB_CUDA_TRY(cudaFuncSetAttribute(tile_kernel<T, DP, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<DP>::SMEM));
        NKB_CUDA_TRY(cudaFuncSetAttribute(tile_kernel<T, DP, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<DP>::SMEM));
        return NKB_OK;
      }))
    return s;
  const Args &a = p.a;
  CUtensorMap mq, mk, mv;
  const int64_t d8 = (a.head_dim + 7) / 8 * 8;
  const uint64_t dims[4] = {(uint64_t)a.head_dim, (uint64_t)p.G, (uint64_t)a.kv_heads, (uint64_t)a.tokens};
  const uint64_t strides[3] = {(uint64_t)(p.G > 1 ? a.q_head : d8), (uint64_t)(a.kv_heads > 1 ? p.G * a.q_head : d8),
                               (uint64_t)(a.tokens > 1 ? a.q_token : d8)};
  const uint32_t box[4] = {64, (uint32_t)p.G, 1, (uint32_t)p.P};
  if (int s = make_bf16_map(&mq, a.q, 4, dims, strides, box)) return s;
  if (int s = cache_map(&mk, a.k_cache, a, a.k_page, a.k_slot, a.k_cache_head)) return s;
  if (int s = cache_map(&mv, a.v_cache, a, a.v_page, a.v_slot, a.v_cache_head)) return s;
  const bool listed = p.own && !p.inside;
  if (listed) {
    pairs_kernel<<<1, SCHED, 0, st>>>(p);
    if (int s = launch_status("paged pairs")) return s;
  }
  NKB_CUDA_TRY(launch_pdl(listed, p.inside ? tile_kernel<T, DP, true> : tile_kernel<T, DP, false>, dim3(p.max_ctas),
                          dim3(THREADS), Cfg<DP>::SMEM, st, mq, mk, mv, p));
  if (int s = launch_status("paged_tile")) return s;
  // nothing to join where the tokens alone make enough units for them to stay whole
  const int64_t per = 2 * p.P, units = (a.tokens + per - 1) / per * a.kv_heads;
  if (p.keep || p.max_ctas < 2 || units >= (int64_t)WHOLE * p.max_ctas) return NKB_OK;
  NKB_CUDA_TRY(launch_pdl(true, tile_join_kernel<T, DP>, dim3((p.max_ctas - 1) * (2 * BM / 32)), dim3(JOIN), 0, st, p));
  return launch_status("paged_tile join");
}

}  // namespace

bool tile_form(const Args &a) {
  return a.dtype != NKB_F32 && a.head_dim <= 128 && a.q_heads / a.kv_heads <= BM && a.page_size >= 8 &&
         log2_of(a.page_size) >= 0 && a.pages > 0;
}

bool tile_strides(const Args &a) {
  if (!aligned16(a)) return false;
  // a broadcast axis (stride 0) has no tensor map
  return (a.page_size == 1 || (a.k_slot > 0 && a.v_slot > 0)) && (a.kv_heads == 1 || (a.k_cache_head > 0 && a.v_cache_head > 0)) &&
         (a.pages == 1 || (a.k_page > 0 && a.v_page > 0)) && (a.q_heads == 1 || a.q_head > 0) && (a.tokens == 1 || a.q_token > 0);
}

size_t tile_workspace(const Args &a, int device, bool own, bool prefix, bool keep) {
  return layout(a, num_sms(device), own, prefix, keep).bytes;
}

int tile_params(const Args &a, int device, void *workspace, bool own, bool prefix, bool keep, Params *p) {
  p->a = a;
  p->G = (int)(a.q_heads / a.kv_heads);
  p->P = BM / p->G;
  p->page_shift = log2_of(a.page_size);
  p->max_ctas = num_sms(device);
  p->own = own;
  p->prefix = prefix;
  p->keep = keep;
  p->scale_log2 = (float)(a.scale * LOG2E);
  p->wide = reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.out_token % 16 == 0 && a.out_head % 16 == 0;
  const Layout x = layout(a, p->max_ctas, own, prefix, keep);
  p->max_pairs = x.max_pairs;
  // (more units than CTAs may be handed out one by one, by a counter that the list's kernel sets)
  p->inside = own && x.max_pairs <= LIST && a.seqs <= LIST && x.max_pairs * a.kv_heads <= p->max_ctas;
  char *w = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(workspace) + WS_ALIGN - 1) / WS_ALIGN * WS_ALIGN);
  p->head = reinterpret_cast<int64_t *>(w);
  p->next = reinterpret_cast<int *>(w + x.next);
  p->pairs = reinterpret_cast<Pair *>(w + x.pairs);
  p->seq_pairs = reinterpret_cast<int *>(w + x.seqs);
  p->ws = reinterpret_cast<float *>(w + x.ws);
  return NKB_OK;
}

int tile_launch(const Params &p, cudaStream_t st, int device) {
  if (p.a.dtype == NKB_BF16)
    return p.a.head_dim <= 64 ? launch<__nv_bfloat16, 64>(p, st, device) : launch<__nv_bfloat16, 128>(p, st, device);
  return p.a.head_dim <= 64 ? launch<__half, 64>(p, st, device) : launch<__half, 128>(p, st, device);
}

int tile_read_and_clear_error(int *flag) {
  int zero = 0;
  NKB_CUDA_TRY(cudaMemcpyFromSymbol(flag, g_tile_error, sizeof(int)));
  if (*flag) NKB_CUDA_TRY(cudaMemcpyToSymbol(g_tile_error, &zero, sizeof(int)));
  return NKB_OK;
}

}  // namespace pattn
}  // namespace nkb
