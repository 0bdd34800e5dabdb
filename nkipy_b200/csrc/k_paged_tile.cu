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
// the device: a small kernel lists the pairs first.
//
// Warps of a CTA:
//   8      producer: TMA loads of Q (both tiles) and, page by page, of K and V
//          into rings of stages that are released separately;
//   9      one thread issues the products, in the order S_A(0) S_B(0), then per
//          block PV_A(c) S_A(c+1) PV_B(c) S_B(c+1), so one tile's softmax
//          overlaps the other's products; it owns the TMEM;
//   10     walks the CTA's share and hands its segments to the others through a
//          small ring, ahead of them;
//   0-3, 4-7  softmax of tile A and of tile B, one thread per row: scores from
//          TMEM, mask, running maximum (raised only when it grows by more than
//          2^8, O is then scaled in TMEM), exp2, P as 16-bit pairs over the
//          scores, handed over in two halves; at a segment's end O / l to
//          memory, or the partial.
// Keys that no row of the CTA sees may hold anything (another sequence's rows,
// infinities, NaN): their scores are replaced; pages of which no key is seen are
// not read (TMA fills zeros), and the unseen V rows of the others are set to
// zero in shared memory before the product that would multiply them by zero.
// TMEM: S_A S_B O_A O_B, 128 columns each.  Every wait is bounded.
#include "paged_attn.cuh"
#include "sm100.cuh"

namespace nkb {
namespace pattn {
namespace {

using namespace sm100;

using namespace several;

constexpr int W_PROD = 8, W_MMA = 9, W_WALK = 10, THREADS = 384;
// registers: 168 a thread at launch, moved from the last four warps to the
// softmax warps (8 x 208 + 4 x 88 = 12 x 168)
constexpr int REGS_SOFTMAX = 208, REGS_REST = 88;
constexpr int RING = 4;  // segments
constexpr int HALF = 128 * 64 * 2;  // 128 rows x 64 columns, 128-byte swizzle
constexpr uint32_t T_S = 0, T_O = 256, TMEM_COLS = 512;
constexpr float RESCALE = 8.f;  // log2 headroom before the running maximum is raised

__device__ int g_tile_error = 0;

template <int DP>
struct Cfg {
  static constexpr int HALVES = DP / 64, TILE = HALVES * HALF, STAGES = DP == 128 ? 2 : 4;
  static constexpr int OFF_K = 2 * TILE, OFF_V = OFF_K + STAGES * TILE, OFF_BAR = OFF_V + STAGES * TILE;
  static constexpr int OFF_ITEMS = OFF_BAR + 320;
  static constexpr int SMEM = 1024 + OFF_ITEMS + RING * 64;
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
  int64_t before = 0, all = 0;
  for (int w = 0; w < SCHED / 32; ++w) {
    if (w < warp) before += s[w];
    all += s[w];
  }
  *total = all;
  return before + x - v;
}

// tokens of list entry i: those before the sequences, sequence i - 1, those after
__device__ __forceinline__ void tokens_of(const Args &a, int i, int &first, int &n) {
  const int B = (int)a.seqs, T = (int)a.tokens;
  const int lo = i == 0 ? 0 : a.q_start[i - 1], hi = i > B ? T : a.q_start[i];
  first = max(0, min(lo, T));
  n = max(0, min(hi, T) - first);
}

__global__ void __launch_bounds__(SCHED) pairs_kernel(const __grid_constant__ Params p) {
  const Args &a = p.a;
  const int per = 2 * p.P, B = (int)a.seqs, T = (int)a.tokens;
  const int lists = p.own ? B + 2 : 0, front = p.prefix ? (T + per - 1) / per : 0;
  pdl_trigger();
  int64_t npairs = front;
  for (int base = 0; base < lists; base += SCHED) {
    const int i = base + threadIdx.x;
    int first, n = 0;
    if (i < lists) tokens_of(a, i, first, n);
    int64_t all;
    const int64_t at = npairs + block_scan((n + per - 1) / per, &all);
    if (i < lists) p.seq_pairs[i] = (int)min(at, (int64_t)p.max_pairs);
    npairs += all;
  }
  // the list holds max_pairs: q_start entries that overlap, which no caller means, would need more
  const int U = (int)min(npairs, (int64_t)p.max_pairs);
  __syncthreads();
  int64_t blocks = 0;
  for (int base = 0; base < U; base += SCHED) {
    const int u = base + threadIdx.x;
    int64_t nb = 0;
    Pair x = {-2, 0, 0, 0};
    if (u < front) {
      x = {-1, u * per, min(per, T - u * per), 0};
    } else if (u < U) {
      int lo = 0, hi = lists - 1;  // the last list that begins at or before u
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (p.seq_pairs[mid] <= u) lo = mid;
        else hi = mid - 1;
      }
      int first, n;
      tokens_of(a, lo, first, n);
      const int off = (u - p.seq_pairs[lo]) * per;
      x.tok0 = first + off;
      x.ntok = max(0, min(per, n - off));
      if (lo >= 1 && lo <= B) {
        x.seq = lo - 1;
        x.pos0 = a.kv_len[lo - 1] - n + off;
      }
    }
    if (u < U) {
      nb = blocks_of(p, x).n;
      p.pairs[u] = x;
    }
    int64_t all;
    const int64_t at = blocks + block_scan(nb, &all);
    if (u < U) p.head[1 + u] = at;
    blocks += all;
  }
  if (threadIdx.x == 0) {
    p.head[0] = U;
    p.head[1 + U] = blocks;
  }
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

// A segment as the roles need it.
struct Item {
  int seq, tok0, ntok, pos0, hk;
  int end, low, ns, w0;  // Blocks
  int k0, n;             // first block, number of blocks; n = 0: the share is done
  int nb[2];             // blocks that each tile needs
  int final, slot;
};

template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

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
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

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

template <class T, int DP>
__global__ void __launch_bounds__(THREADS, 1)
    tile_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                const __grid_constant__ CUtensorMap mv, const __grid_constant__ Params p) {
  using C = Cfg<DP>;
  constexpr int ST = C::STAGES;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::OFF_BAR);
  uint64_t *q_full = bars, *q_empty = bars + 1, *s_full = bars + 2, *p_half = bars + 4, *p_ready = bars + 6,
           *o_done = bars + 8, *o_free = bars + 10, *i_full = bars + 12, *i_empty = i_full + RING, *k_full = i_empty + RING,
           *k_empty = k_full + ST, *v_full = k_empty + ST, *v_empty = v_full + ST;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(v_empty + ST);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  Item *ring = reinterpret_cast<Item *>(smem + C::OFF_ITEMS);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const Args &a = p.a;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_half[t], BM);
      mbar_init(&p_ready[t], BM);
      mbar_init(&o_done[t], 1);
      mbar_init(&o_free[t], BM);
    }
    for (int s = 0; s < RING; ++s) {
      mbar_init(&i_full[s], 1);
      mbar_init(&i_empty[s], 10);  // producer, issuer, eight softmax warps
    }
    for (int s = 0; s < ST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
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
  // the next segment, from the ring (whole warps, or one thread for the issuer)
  auto take = [&](Item &x, bool whole_warp) {
    const int i = items % RING;
    ok = whole_warp ? wait_warp(&i_full[i], (items / RING) & 1, abort_flag) : wait(&i_full[i], (items / RING) & 1, abort_flag);
    if (!ok) return false;
    x = ring[i];
    if (whole_warp) __syncwarp();
    if (!whole_warp || lane == 0) mbar_arrive(&i_empty[i]);
    ++items;
    return x.n > 0;
  };
  auto block_of = [](const Item &x, int i) { return i < x.ns ? i : x.w0 + i - x.ns; };

  if (warp >= W_PROD) {
    regs_dec<REGS_REST>();
    if (warp == W_WALK) {
      // ---------------- segments of this CTA's share ----------------
      Walk walk(p, blockIdx.x);
      Segment s;
      while (true) {
        const bool more = walk.next(s, lane);
        const int i = items % RING;
        if (!wait_warp(&i_empty[i], ((items / RING) & 1) ^ 1, abort_flag)) break;
        if (lane == 0) {
          Item x;
          x.n = 0;
          if (more) {
            x = {s.x.seq, s.x.tok0, s.x.ntok, s.x.pos0, s.hk, s.k.end, s.k.low, s.k.ns, s.k.w0, s.k0, s.k1 - s.k0, {0, 0},
                 s.all && !p.keep, s.slot};
            for (int t = 0; t < 2; ++t) x.nb[t] = max(0, min(x.n, tile_blocks(p, s.x, s.k, t) - s.k0));
          }
          ring[i] = x;
          mbar_arrive(&i_full[i]);
        }
        __syncwarp();
        ++items;
        if (!more) break;
      }
    } else if (warp == W_PROD) {
      // ---------------- TMA producer ----------------
      const int ps = (int)a.page_size, box = min(ps, BN), npb = BN / box;  // pages (or page parts) per block
      uint32_t segs = 0, blk = 0;
      Item x;
      while (ok && take(x, true)) {
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
    } else if (warp == W_MMA && lane == 0) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t ID_S = idesc<T>(128, BN, 0), ID_O = idesc<T>(128, DP, 1);
      const Desc dq(smem_desc(smem_u32(smem), 16, 1024)), dk(smem_desc(smem_u32(smem + C::OFF_K), 16, 1024)),
          dv(smem_desc(smem_u32(smem + C::OFF_V), HALF, 1024));
      uint32_t segs = 0, blk = 0, cnt[2] = {0, 0}, outs[2] = {0, 0};
      Item x;
      while (ok && take(x, false)) {
        const int n = x.n;
        auto qk = [&](int t, int c) {  // S_t = Q_t K_c^T
          const Desc k(dk.at(((blk + c) % ST) * C::TILE)), q(dq.at(t * C::TILE));
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk) {
            const uint32_t off = (kk >> 2) * HALF + (kk & 3) * 32;
            umma_f16(tmem + T_S + t * 128, q.at(off), k.at(off), ID_S, kk > 0);
          }
          umma_commit(&s_full[t]);
        };
        auto pv = [&](int t, int c, int half) {  // O_t += P_t V_c, 64 keys of the block
          const Desc v(dv.at(((blk + c) % ST) * C::TILE));
#pragma unroll
          for (int kk = 0; kk < BN / 32; ++kk) {
            const int k = half * (BN / 32) + kk;
            umma_f16_ts(tmem + T_O + t * 128, tmem + T_S + t * 128 + k * 8, v.at(k * 2048), ID_O, (c > 0 || k > 0) ? 1u : 0u);
          }
        };
        auto k_wait = [&](int c) { return wait(&k_full[(blk + c) % ST], ((blk + c) / ST) & 1, abort_flag); };
        if (!(ok = wait(q_full, segs & 1, abort_flag) && k_wait(0))) break;
        ++segs;
        tc_fence_after();
        for (int t = 0; t < 2; ++t)
          if (x.nb[t] > 0) qk(t, 0);
        umma_commit(&k_empty[blk % ST]);
        if (n == 1) umma_commit(q_empty);
        for (int c = 0; ok && c < n; ++c) {
          const bool more = c + 1 < n;
          if (!(ok = wait(&v_full[(blk + c) % ST], ((blk + c) / ST) & 1, abort_flag) && (!more || k_wait(c + 1)))) break;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (c < x.nb[t]) {
              // half of P of block c is written; before a segment's first product, O of the segment before is read
              if (!(ok = wait(&p_half[t], cnt[t] & 1, abort_flag) &&
                         (c > 0 || outs[t] == 0 || wait(&o_free[t], (outs[t] - 1) & 1, abort_flag))))
                break;
              tc_fence_after();
              pv(t, c, 0);
              if (!(ok = wait(&p_ready[t], cnt[t] & 1, abort_flag))) break;
              tc_fence_after();
              pv(t, c, 1);
              umma_commit(&o_done[t]);
              ++cnt[t];
            }
            if (c + 1 < x.nb[t]) qk(t, c + 1);
          }
          if (!ok) break;
          if (more) {
            umma_commit(&k_empty[(blk + c + 1) % ST]);
            if (c + 2 == n) umma_commit(q_empty);
          }
          umma_commit(&v_empty[(blk + c) % ST]);
        }
        blk += n;
        for (int t = 0; t < 2; ++t) outs[t] += x.nb[t] > 0;
      }
    }
  } else {
    // ---------------- softmax and results: tile t, row r ----------------
    regs_inc<REGS_SOFTMAX>();
    const int t = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t rows = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t s_col = rows + T_S + t * 128, o_col = rows + T_O + t * 128;
    const int g = r % p.G, tok = t * p.P + r / p.G;  // query head in the group, token in the pair
    const uint64_t scale2 = pair2(p.scale_log2, p.scale_log2);
    uint32_t blk = 0, cnt = 0;
    Item x;
    while (ok && take(x, true)) {
      const int nb = x.nb[t];
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
      const int all_first = (int)min(a.sinks, (int64_t)x.end);
      float m = -INFINITY, l = 0.f;  // running (possibly stale) maximum in log2 units, and sum
      for (int c = 0; c < nb; ++c, ++cnt) {
        const int key0 = block_of(x, x.k0 + c) * BN;
        if (!(ok = wait_warp(&s_full[t], cnt & 1, abort_flag))) break;
        tc_fence_after();
        uint32_t v[128];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32_nw(s_col + i * 32, v + i * 32);
        tmem_ld_wait();
        if (__any_sync(0xffffffffu, key0 + BN > hi || (key0 < lo && key0 + BN > first))) {
          // a bit per key: below hi, and from lo or below first
          const int h = hi - key0, w = lo - key0, f = first - key0;
          auto below = [](int n) -> uint32_t { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t bits = below(h - 32 * i) & (~below(w - 32 * i) | below(f - 32 * i));
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (!(bits >> j & 1)) v[32 * i + j] = 0xff800000u;
          }
        }
        if (key0 + BN > x.end || (key0 < x.low && key0 + BN > all_first)) {
          // rows of V that no token of the pair sees: zeros
          const int key = key0 + r;
          const bool unseen = key >= x.end || (key < x.low && key >= all_first);
          if (__any_sync(0xffffffffu, unseen)) {
            const uint32_t b = blk + c;
            if (!(ok = wait_warp(&v_full[b % ST], (b / ST) & 1, abort_flag))) break;
            if (unseen) {
              uint8_t *row = smem + C::OFF_V + (b % ST) * C::TILE + r * 128;
#pragma unroll
              for (int j = 0; j < C::HALVES; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4 *>(row + j * HALF + i * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 128; j += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mx4[i] = max3(mx4[i], __uint_as_float(v[j + 2 * i]), __uint_as_float(v[j + 2 * i + 1]));
        float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        mx = mx == -INFINITY ? -INFINITY : mx * p.scale_log2;
        const bool raise = mx > m + RESCALE;
        if (__any_sync(0xffffffffu, raise)) {
          const float m_new = raise ? mx : m;
          const float alpha = m == -INFINITY ? 0.f : raise ? ex2(m - m_new) : 1.f;
          if (c > 0) {
            if (!(ok = wait_warp(&o_done[t], (cnt - 1) & 1, abort_flag))) break;
            tc_fence_after();
#pragma unroll 1
            for (int i = 0; i < DP / 16; ++i) {
              uint32_t o[16];
              tmem_ld16(o_col + i * 16, o);
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
              tmem_st16(o_col + i * 16, o);
            }
            tmem_st_wait();
          }
          l *= alpha;
          m = m_new;
        }
        const float mm = m == -INFINITY ? 0.f : m;
        const uint64_t base2 = pair2(-mm, -mm);
        uint64_t l2[2] = {0, 0};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int j = half * 64; j < half * 64 + 64; j += 2) {
            float e0, e1;
            unpair2(fma2(pair2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), scale2, base2), e0, e1);
            e0 = ex2(e0);
            e1 = ex2(e1);
            l2[(j >> 1) & 1] = add2(l2[(j >> 1) & 1], pair2(e0, e1));
            v[j / 2] = pack<T>(e0, e1);
          }
          tmem_st16(s_col + half * 32, v + half * 32);
          tmem_st16(s_col + half * 32 + 16, v + half * 32 + 16);
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(half ? &p_ready[t] : &p_half[t]);
        }
        float s0, s1, s2, s3;
        unpair2(l2[0], s0, s1);
        unpair2(l2[1], s2, s3);
        l += (s0 + s1) + (s2 + s3);
      }
      if (!ok) break;
      blk += x.n;
      if (nb > 0) {
        if (!(ok = wait_warp(&o_done[t], (cnt - 1) & 1, abort_flag))) break;
        tc_fence_after();
      }
      const float inv = l > 0.f ? 1.f / l : 0.f;
      const int D = (int)a.head_dim, token = x.tok0 + tok;
      T *dst = static_cast<T *>(a.out) + token * a.out_token + (x.hk * p.G + g) * a.out_head;
      float *part = p.ws + (int64_t)x.slot * C::SLOT;
#pragma unroll 1
      for (int i = 0; i < DP / 32; ++i) {
        uint32_t o[32];
        __syncwarp();  // the warp reads TMEM together
        if (nb > 0) {
          tmem_ld32(o_col + i * 32, o);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0;
        }
        if (row_ok && x.final) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint4 w;
            w.x = pack<T>(__uint_as_float(o[j]) * inv, __uint_as_float(o[j + 1]) * inv);
            w.y = pack<T>(__uint_as_float(o[j + 2]) * inv, __uint_as_float(o[j + 3]) * inv);
            w.z = pack<T>(__uint_as_float(o[j + 4]) * inv, __uint_as_float(o[j + 5]) * inv);
            w.w = pack<T>(__uint_as_float(o[j + 6]) * inv, __uint_as_float(o[j + 7]) * inv);
            if (i * 32 + j < D) *reinterpret_cast<uint4 *>(dst + i * 32 + j) = w;
          }
        } else if (row_ok) {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<uint4 *>(part + (t * BM + r) * DP + i * 32 + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
        }
      }
      if (row_ok && !x.final) *reinterpret_cast<float2 *>(part + 2 * BM * DP + 2 * (t * BM + r)) = make_float2(m, l);
      __syncwarp();
      if (nb > 0) {
        tc_fence_before();
        mbar_arrive(&o_free[t]);
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

// Joins the partials of the units that a share's end cuts: block (c, y) looks at
// the unit cut by the beginning of CTA c's share, and takes 32 of its rows if
// that is the unit's first cut.
template <class T, int DP>
__global__ void __launch_bounds__(256) tile_join_kernel(const __grid_constant__ Params p) {
  using C = Cfg<DP>;
  pdl_wait();
  const Args &a = p.a;
  const Walk walk(p, 0);
  const int c = blockIdx.x + 1;
  if (c >= walk.ctas) return;
  const int64_t cut = share(walk.total, c, walk.ctas);
  Segment s;
  walk.locate(cut, s, threadIdx.x % 32);
  const int64_t first = cut - s.k0;
  if (s.k0 == 0) return;  // the share begins with the unit
  const Parts parts = parts_of(walk.total, first, s.k.n, p.max_ctas, 0);
  if (parts.c0 != c - 1) return;
  const int D = (int)a.head_dim;
  for (int i = threadIdx.x; i < 32 * (DP / 4); i += 256) {
    const int row = blockIdx.y * 32 + i / (DP / 4), d = i % (DP / 4) * 4, t = row / BM, r = row % BM;
    const int g = r % p.G, tok = t * p.P + r / p.G;
    if (r >= p.P * p.G || tok >= s.x.ntok || d >= D) continue;
    auto slot = [&](int j) { return p.ws + (int64_t)parts.slot(j) * C::SLOT; };
    float M = -INFINITY, L = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < parts.n; ++j) M = fmaxf(M, __ldcg(slot(j) + 2 * BM * DP + 2 * row));
    for (int j = 0; j < parts.n; ++j) {
      const float2 ml = __ldcg(reinterpret_cast<const float2 *>(slot(j) + 2 * BM * DP + 2 * row));
      const float4 y = __ldcg(reinterpret_cast<const float4 *>(slot(j) + row * DP + d));
      const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
      L += ml.y * f;
      x[0] += y.x * f;
      x[1] += y.y * f;
      x[2] += y.z * f;
      x[3] += y.w * f;
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + (s.x.tok0 + tok) * a.out_token + (s.hk * p.G + g) * a.out_head + d) =
        make_uint2(pack<T>(x[0] * inv, x[1] * inv), pack<T>(x[2] * inv, x[3] * inv));
  }
}

int log2_of(int64_t x) {
  int s = 0;
  while ((int64_t(1) << s) < x) ++s;
  return (int64_t(1) << s) == x ? s : -1;
}

// workspace: head | pairs | seq_pairs | partial slots
struct Layout {
  size_t pairs, seqs, ws, bytes;
  int max_pairs;
};
Layout layout(const Args &a, int max_ctas, bool own, bool prefix, bool keep) {
  const int64_t per = 2 * (BM / (a.q_heads / a.kv_heads)), T = a.tokens;
  Layout x;
  // every sequence, and the tokens before and after them, may end in a part of a pair
  x.max_pairs = (int)((prefix ? (T + per - 1) / per : 0) + (own ? T / per + a.seqs + 2 : 0));
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  x.pairs = up(((size_t)x.max_pairs + 2) * 8);
  x.seqs = x.pairs + up((size_t)x.max_pairs * sizeof(Pair));
  x.ws = x.seqs + up((size_t)(own ? a.seqs + 2 : 0) * 4);
  const size_t slot = (a.head_dim <= 64 ? Cfg<64>::SLOT : Cfg<128>::SLOT) * sizeof(float);
  x.bytes = x.ws + (2 * (size_t)max_ctas + (keep ? (size_t)x.max_pairs * a.kv_heads : 0)) * slot;
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
        NKB_CUDA_TRY(cudaFuncSetAttribute(tile_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<DP>::SMEM));
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
  pairs_kernel<<<1, SCHED, 0, st>>>(p);
  if (int s = launch_status("paged pairs")) return s;
  NKB_CUDA_TRY(launch_pdl(true, tile_kernel<T, DP>, dim3(p.max_ctas), dim3(THREADS), Cfg<DP>::SMEM, st, mq, mk, mv, p));
  if (int s = launch_status("paged_tile")) return s;
  if (p.keep || p.max_ctas < 2) return NKB_OK;
  NKB_CUDA_TRY(launch_pdl(true, tile_join_kernel<T, DP>, dim3(p.max_ctas - 1, 2 * BM / 32), dim3(256), 0, st, p));
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
  p->scale_log2 = (float)(a.scale * 1.4426950408889634);
  const Layout x = layout(a, p->max_ctas, own, prefix, keep);
  p->max_pairs = x.max_pairs;
  char *w = static_cast<char *>(workspace);
  p->head = reinterpret_cast<int64_t *>(w);
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
