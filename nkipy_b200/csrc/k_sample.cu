// Draws one token per row of logits: temperature, top-k, top-p and min-p, then
// the inverse of the kept weights' running sum at u.
//
// Weights are w = floor(2^32 exp((x - max) / temperature)): whole numbers, so
// every sum below is exact and independent of its order, whatever the number
// of threads.  A logit's key is the order-preserving image of its fp32 value
// (-0 as +0, NaN as -inf); elements are ordered by their rank word, the key
// above the complement of the index, so equal logits rank by index and the
// kept set is "rank word >= threshold", with e >= min_p.
//
// A cluster of up to 8 CTAs holds a row in its shared memory: the logits are read
// from memory once.  What bounds the kernel is then waiting: shared memory lets two CTAs
// of 8 warps on an SM, which issue in 24 % of the cycles (128 mixed rows), through
// the cluster's meetings (about a microsecond each), shared memory's latency and short
// serial steps; 128 rows of 4 CTAs are 1.7 waves besides.  So each way of filtering has
// the fewest meetings it can (GPU times for 1 row of 32000 fp32, and 128 rows of 151936
// bf16, whose 39 MB a copy reads in 6 us):
//   greedy  the CTAs' maxima: one meeting; 3 and 16 us
//   top-k   of up to FAST_K: the CTAs' largest thread maxima bound the row's k-th
//           largest element; what passes (two to three k elements) goes to one CTA,
//           which sorts it, applies the other filters and draws alone: three; 10 and
//           35 us for k = 50
//   top-p, other top-k   a histogram of counts and exact weights over 512 bins
//           linear in (max - x) / temperature, summed over the cluster (again
//           within the threshold's bin if that holds too many); the elements of
//           the threshold's bin go to every CTA, which narrows them down and sorts
//           the last few: five (more for both); 20 and 145 us for p = 0.95
//   none    the kept weight of each warp, whose part of the row is contiguous; the
//           warp in which the running sum passes u times the total walks its part:
//           two; 6 and 47 us
// Where that does not do (thousands of equal logits at a threshold) the threshold
// is found bit by bit over the cluster.

#include <cooperative_groups.h>

#include <type_traits>

#include "paged.cuh"

namespace nkb {
namespace sample {

namespace cg = cooperative_groups;
using Args = nkb_sample_args;
using u64 = unsigned long long;

__device__ __forceinline__ float load_x(const void *p, int64_t i, int dt) {
  float x = __uint_as_float(load_as_reg(p, i, dt));
  if (x != x) x = -INFINITY;
  return x + 0.f;  // -0 becomes +0
}
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t KEY_NEG_INF = 0x007fffffu, KEY_POS_INF = 0xff800000u;  // key_of(-inf), key_of(inf)
constexpr int IDX_BITS = 21;
constexpr int64_t MAX_VOCAB = 1 << IDX_BITS;
__device__ __forceinline__ u64 rank_word(uint32_t key, int idx) {
  return ((u64)key << IDX_BITS) | (uint32_t)(MAX_VOCAB - 1 - idx);
}

// The softmax's terms: each step is rounded to fp32 as the definition says, so that
// the drawn token is the definition's.  (One product by log2(e) / temperature and the
// power-of-two unit took 76 us instead of 84 for 128 mixed rows of 151936 entries, and
// in some batches one row drew a neighbour of its token.)
struct Row {
  float max, inv;  // largest logit, 1 / temperature
  __device__ __forceinline__ Row(float max, float temperature) : max(max), inv(fminf(1.f / temperature, 3.4028235e38f)) {}
  __device__ __forceinline__ float t(float x) const { return __fmul_rn(__fsub_rn(x, max), inv); }
  __device__ __forceinline__ float e(float x) const { return x == max ? 1.f : x == -INFINITY ? 0.f : expf(t(x)); }
  // floor(2^32 e) for e in [0, 1]: the significand, moved (0 for NaN)
  static __device__ __forceinline__ u64 w(float e) {
    const uint32_t b = __float_as_uint(e);
    const uint32_t low = __funnelshift_rc((b << 8) | 0x80000000u, 0, 126 - (b >> 23));
    return ((u64)(b == 0x3f800000u) << 32) | low;  // e = 1 alone has bit 32, and no lower bits
  }
  // weight of a logit, where max is finite: without branches (0 for -inf and NaN)
  __device__ __forceinline__ u64 weight(float x) const { return w(expf(t(x))); }
};

// floor(p * total) for p in [0, 1), exactly: total times the significand, moved.
__device__ __forceinline__ u64 part_of(float p, u64 total) {
  const uint32_t b = __float_as_uint(p), e = b >> 23;
  const u64 m = (b & 0x7fffffu) | 0x800000u, lo = total * m, hi = __umul64hi(total, m);
  const uint32_t down = 150 - e;  // from 24; total * m < 2^77
  return !(p > 0.f) || down >= 77 ? 0 : down >= 64 ? hi >> (down - 64) : (hi << (64 - down)) | (lo >> down);
}
// The weight that top-p asks for: one at least.
__device__ __forceinline__ u64 share_of(float p, u64 total) { return max((u64)1, part_of(p, total)); }
// The random place among `total`.
__device__ __forceinline__ u64 place(float u, u64 total) { return u >= 1.f ? total - 1 : part_of(u, total); }

// ---- rows in a cluster's shared memory -------------------------------------
constexpr int NT = 256, NW = NT / 32, MAX_C = 8;
constexpr int CAP = 2048;         // elements that a CTA lists
constexpr int FEW = 256;          // elements that are sorted one a thread
// Top-k that one CTA sorts: some 2 k to 3 k candidates are expected, CAP fit.  Sorted
// and by histogram, us, with top-p 0.9 behind it: k = 200, 1 row of 32000 16 / 20, 128
// of 151936 48 / 108; k = 256 17 / 22 and 54 / 110 (without top-p 17 / 16 and 54 / 94).
constexpr int FAST_K = 256;
constexpr int MAX_SLICE = 65528;  // elements per CTA: their low halves' sum stays in 32 bits
constexpr int BINS = 512, QN = BINS * BINS;  // bins, and the finest ones, linear in (max - x) / temperature
constexpr float SPAN = 22.25f;    // e^-SPAN < 2^-32

constexpr int OWN = 3 * BINS / 2; // elements that a CTA gives to the list

struct Shared {
  u64 list[CAP], few[FEW], weights[FAST_K];
  u64 row_w[BINS];                                        // weights per bin, whole row
  u64 warp_sums[MAX_C][NW], sums[2][MAX_C], part_red[NW][16], red[NW], out[2];
  uint32_t row_c[BINS];                                   // counts
  union {
    struct {
      uint32_t hc[BINS], hl[BINS], hh[BINS];              // this CTA's counts and halves of the weights
    };
    u64 own[OWN];                                         // its elements of one bin, afterwards
  };
  float maxima[MAX_C];
  int counts[2][MAX_C], found[MAX_C], bounds[2], n_list, n_own, n_few, bin;
};

template <class V, class Op>
__device__ __forceinline__ V reduce(V v, Op op, V *shared) {  // over the block, to every thread
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int w = 16; w; w >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, w));
  __syncthreads();  // earlier readers of `shared` are done
  if (lane == 0) shared[warp] = v;
  __syncthreads();
  v = shared[lane % NW];
#pragma unroll
  for (int w = NW / 2; w; w >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, w));
  return v;
}
__device__ __forceinline__ u64 add64(u64 x, u64 y) { return x + y; }

// The steps below run once or twice a row: code that is shared is fetched once.
__device__ __noinline__ u64 block_total(Shared &s, u64 v) { return reduce(v, add64, s.red); }

// Exclusive sum over the block's threads; *total gets the sum.
__device__ __noinline__ u64 scan(Shared &s, u64 v, u64 *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 x = v;
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, x, w);
    if (lane >= w) x += y;
  }
  __syncthreads();
  if (lane == 31) s.red[warp] = x;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < warp) before += s.red[w];
    all += s.red[w];
  }
  *total = all;
  return before + x - v;
}

// First bin in which the running sum of get(bin) reaches `target` (-1: none),
// to every thread; the sum before it in s.out[0].
template <int N, class Get>
__device__ __forceinline__ int crossing(Shared &s, u64 target, Get get) {
  constexpr int PER = N / NT;
  const int tid = threadIdx.x;
  u64 v[PER], own = 0, all;
#pragma unroll
  for (int i = 0; i < PER; ++i) own += v[i] = get(tid * PER + i);
  if (tid == 0) s.bin = -1;
  u64 before = scan(s, own, &all);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (before < target && target <= before + v[i]) {
      s.bin = tid * PER + i;
      s.out[0] = before;
    }
    before += v[i];
  }
  __syncthreads();
  return s.bin;
}

// Lowest key in (-inf, inf] that `yes` holds for, where it holds for `top` and
// for every key above one it holds for: by one warp, first the 32 keys around a
// guess, then 32 pivots at a time.
template <class Yes>
__device__ __forceinline__ uint32_t lowest_key(uint32_t top, float guess, Yes yes) {
  uint32_t lo = KEY_NEG_INF, hi = top;  // not at lo, at hi
  const int lane = threadIdx.x & 31;
  const uint32_t g = key_of(guess);
  const uint32_t base = g > KEY_NEG_INF + 16 && g < top ? g - 16 : KEY_NEG_INF;
  uint32_t step = 1, from = base;
  while (true) {
    const uint32_t off = step * (lane + 1), at = off < hi - from ? from + off : hi;
    const uint32_t m = __ballot_sync(0xffffffffu, yes(of_key(at)));
    const int f = __ffs(m) - 1;  // first pivot it holds for
    if (f < 0) {
      lo = from + 32 * step;  // (only around the guess: else the last pivot is hi)
    } else {
      const uint32_t up = step * (f + 1);
      const uint32_t was = from;
      if (up < hi - from) hi = from + up;
      if (f > 0) lo = was + step * f;
    }
    if (hi - lo <= 1) return hi;
    from = lo;
    step = (hi - lo - 1) / 32 + 1;
  }
}

// Fine bin of a logit, and the lowest logit of the bins up to q (NaN, which no
// logit is at or above, for q < 0).
__device__ __forceinline__ int bin_of(const Row &f, float x) { return min(QN - 1, (int)__fmul_rn(f.t(x), -(float)QN / SPAN)); }
__device__ __noinline__ float edge_of(const Row &f, int q) {
  if (q < 0) return __uint_as_float(0x7fc00000u);
  return of_key(lowest_key(key_of(f.max), f.max - (float)(q + 1) * (SPAN / QN) / f.inv, [&](float x) { return bin_of(f, x) <= q; }));
}

// Sorts list[0, n), n <= CAP, largest first (a bitonic network, padded with zeros
// to a power of two).
__device__ void sort_down(u64 *list, int n) {
  int N = 64;
  while (N < n) N *= 2;
  for (int i = n + threadIdx.x; i < N; i += NT) list[i] = 0;
  __syncthreads();
  for (int size = 2; size <= N; size *= 2)
    for (int stride = size / 2; stride; stride /= 2) {
#pragma unroll
      for (int m = 0; m < CAP / 2 / NT; ++m) {
        const int q = threadIdx.x + m * NT;
        if (q >= N / 2) break;
        const int i = 2 * q - (q & (stride - 1)), j = i + stride;
        const u64 x = list[i], y = list[j];
        if ((x < y) == ((i & size) == 0)) {
          list[i] = y;
          list[j] = x;
        }
      }
      // while the stride is at most 32, the next one's elements are this warp's own
      if (stride > 1 && stride <= 32) __syncwarp();
      else __syncthreads();
    }
}

// Sorts the values of the block's first n threads, largest first (the others have 0).
__device__ __noinline__ void sort_down_few(u64 *shared, u64 &v, int n) {
  static_assert(FEW == NT, "one a thread");
  const int i = threadIdx.x;
#pragma unroll 1
  for (int size = 2; size < 2 * n; size *= 2)
#pragma unroll 1
    for (int stride = size / 2; stride; stride /= 2) {
      u64 other;
      if (stride < 32) {
        other = __shfl_xor_sync(0xffffffffu, v, stride);
      } else {
        __syncthreads();
        shared[i] = v;
        __syncthreads();
        other = shared[i ^ stride];
      }
      const bool first = (i & stride) == 0, down = (i & size) == 0;
      v = (first == down) == (other > v) ? other : v;
    }
}

// The rest of a row whose n candidates (rank words in s.list) hold its k largest
// elements, by one CTA.
__device__ void draw_sorted(Shared &s, const Args &a, int64_t r, const Row &f, int n, int k, float p, uint32_t key_pmin) {
  const int tid = threadIdx.x;
  if (n <= FEW) {
    u64 v = tid < n ? s.list[tid] : 0;
    sort_down_few(s.few, v, n);
    __syncthreads();
    s.list[tid] = v;
    __syncthreads();
  } else {
    sort_down(s.list, n);
  }
  const int m = min(k, n);
  static_assert(FAST_K <= NT, "one of the k largest a thread");
  uint32_t key = 0;
  u64 w = 0, W;
  if (tid < m) {
    key = (uint32_t)(s.list[tid] >> IDX_BITS);
    w = Row::w(f.e(of_key(key)));
  }
  const u64 before = scan(s, w, &W), T = p < 1.f ? share_of(p, W) : ~0ull;
  s.weights[tid] = tid < m && before < T && key >= key_pmin ? w : 0;
  __syncthreads();
  if (tid >= m) return;
  const u64 own = s.weights[tid], index = s.list[tid] & (MAX_VOCAB - 1);
  u64 total = 0, upto = 0;  // of all, and of those up to this one in index order
  for (int i = 0; i < m; ++i) {
    const u64 x = s.weights[i];
    total += x;
    if ((s.list[i] & (MAX_VOCAB - 1)) >= index) upto += x;
  }
  const u64 at = place(a.u[r], total);
  if (own && upto > at && upto - own <= at) a.tokens[r] = (int)(MAX_VOCAB - 1 - index);
}

template <class T>
struct Slice {  // a CTA's part of a row, in shared memory
  static constexpr int VEC = 16 / sizeof(T);
  const uint4 *xv;
  int i0, v0, v1;  // first index; this warp's vectors
  __device__ static __forceinline__ float get(const uint4 &q, int j) {
    const uint32_t w = (&q.x)[j / (VEC / 4)];
    float x;
    if constexpr (sizeof(T) == 4) x = __uint_as_float(w);
    else if constexpr (std::is_same<T, __half>::value) x = __half2float(__ushort_as_half((unsigned short)(j & 1 ? w >> 16 : w)));
    else x = __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
    return x + 0.f;
  }
  __device__ static __forceinline__ float top(const uint4 &q) {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < VEC; ++j) m = fmaxf(m, get(q, j));  // NaN is passed over
    return m;
  }
  // f(x, index of the first) for this warp's vectors (FEW: those that have an element from `cut` up)
  template <bool FEW, class F>
  __device__ __forceinline__ void vectors(float cut, F f) const {
    for (int v = v0 + (threadIdx.x & 31); v < v1; v += 32) {
      const uint4 q = xv[v];
      if (FEW && !(top(q) >= cut)) continue;
      float x[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] = get(q, j);
      f(x, i0 + v * VEC);
    }
  }
  // the same for the vectors that have an element in [from, to)
  template <class F>
  __device__ __forceinline__ void between(float from, float to, F f) const {
    vectors<true>(from, [&](const float (&x)[VEC], int first) {
      bool any = false;
#pragma unroll
      for (int j = 0; j < VEC; ++j) any |= x[j] >= from && !(x[j] >= to);
      if (any) f(x, first);
    });
  }
  // f(x, index) for this warp's elements from `cut` up (never NaN), where they are few
  template <class F>
  __device__ __forceinline__ void each(float cut, F f) const {
    vectors<true>(cut, [&](const float (&x)[VEC], int first) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (x[j] >= cut) f(x[j], first + j);
    });
  }
};

// The largest rank word that `target` elements (count) or a weight of `target`
// reach, among the elements with rank words from `least`; *mass: the weight from
// it up.  Bit by bit, every CTA of the cluster together.
template <class T, int C>
__device__ __noinline__ u64 find_slowly(Shared &s, const Slice<T> &x, const Row &f, float cut, bool count, u64 target,
                                        u64 least, u64 *mass) {
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  int turn = 0;
  cluster.sync();  // the sums, which are used for other things before, are read
  auto measure = [&](u64 from, bool by_count) {
    u64 sum = 0;
    x.each(cut, [&](float y, int i) {
      const u64 word = rank_word(key_of(y), i);
      if (word >= from && word >= least) sum += by_count ? 1 : f.weight(y);
    });
    sum = reduce(sum, add64, s.red);
    // a CTA can be one turn ahead of another, not two
    if (threadIdx.x < C) cluster.map_shared_rank(s.sums[turn & 1], threadIdx.x)[rank] = sum;
    cluster.sync();
    u64 all = 0;
    for (int c = 0; c < C; ++c) all += s.sums[turn & 1][c];
    ++turn;
    return all;
  };
  u64 word = 0;
  if (measure(0, count) > target || !count) {
    for (int bit = 52; bit >= 0; --bit)
      if (measure(word | (1ull << bit), count) >= target) word |= 1ull << bit;
  }
  *mass = measure(word, false);
  cluster.sync();  // the sums are read
  return word;
}

template <class T, int C>
__global__ void __launch_bounds__(NT, 2) cluster_kernel(const __grid_constant__ Args a, int slice) {
  using X = Slice<T>;
  constexpr int VEC = X::VEC;
  extern __shared__ __align__(16) uint8_t smem[];
  Shared &s = *reinterpret_cast<Shared *>(smem);
  T *xs = reinterpret_cast<T *>(smem + (sizeof(Shared) + 15) / 16 * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // another CTA's shared memory may be touched once all have begun: waited for below
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int64_t r = blockIdx.x / C;
  const int V = (int)a.vocab, i0 = rank * slice, n = max(0, min(slice, V - i0));
  const T *row = static_cast<const T *>(a.logits) + r * a.row_stride + i0;
  // vectors of this warp: contiguous, [v0, v1)
  const int nv = (n + VEC - 1) / VEC, per = (nv + NW - 1) / NW;
  const X x{reinterpret_cast<const uint4 *>(xs), i0, min(nv, warp * per), min(nv, (warp + 1) * per)};

  // logits to shared memory, two maxima a thread; the tail of the last vector is -inf
  float m0 = -INFINITY, m1 = -INFINITY;
  const int full = (reinterpret_cast<uintptr_t>(row) & 15) == 0 ? n / VEC : 0;  // vectors that can be read as such
  constexpr int U = 5;
  for (int v = tid; v < full; v += U * NT) {
    uint4 q[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (v + i * NT < full) q[i] = __ldcs(reinterpret_cast<const uint4 *>(row) + v + i * NT);
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (v + i * NT < full) {
        reinterpret_cast<uint4 *>(xs)[v + i * NT] = q[i];
        float &m = i & 1 ? m1 : m0;
        m = fmaxf(m, X::top(q[i]));
      }
  }
  if (full < nv) {
#pragma unroll 4
    for (int i = full * VEC + tid; i < nv * VEC; i += NT) xs[i] = i < n ? row[i] : (T)(-INFINITY);
    __syncthreads();
    for (int v = full + tid; v < nv; v += NT) m0 = fmaxf(m0, X::top(x.xv[v]));
  }
  for (int i = tid; i < BINS; i += NT) s.hc[i] = s.hl[i] = s.hh[i] = 0;
  if (tid == 0) s.n_list = s.n_own = 0;
  {
    const float m = reduce(fmaxf(m0, m1), [](float x, float y) { return fmaxf(x, y); }, reinterpret_cast<float *>(s.red));
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid < C) cluster.map_shared_rank(s.maxima, tid)[rank] = m;
  }
  cluster.sync();
  float gmax = -INFINITY;
  int owner = 0;  // lowest rank that has the maximum
#pragma unroll
  for (int c = C - 1; c >= 0; --c)
    if (s.maxima[c] >= gmax) {
      gmax = s.maxima[c];
      owner = c;
    }
  if (gmax == -INFINITY) {
    if (rank == 0 && tid == 0) a.tokens[r] = -1;
    return;
  }
  const float temp = a.temperature ? a.temperature[r] : 1.f;
  if (!(temp > 0.f)) {
    if (rank != owner) return;
    u64 first = V;
    x.each(gmax, [&](float, int i) { first = min(first, (u64)i); });
    first = reduce(first, [](u64 x, u64 y) { return x < y ? x : y; }, s.red);
    if (tid == 0) a.tokens[r] = (int)first;
    return;
  }

  if (gmax == INFINITY) {  // only the infinite logits have a weight, all the same: ones among -infinities
    for (int i = tid; i < nv * VEC; i += NT) xs[i] = (float)xs[i] == INFINITY ? (T)1.f : (T)(-INFINITY);
    gmax = 1.f;
    m0 = fmaxf(m0, m1) == INFINITY ? 1.f : -INFINITY;
    m1 = -INFINITY;
    __syncthreads();
  }
  const Row f(gmax, temp);
  const uint32_t kmax = key_of(gmax);
  auto bin = [&](float x) { return bin_of(f, x); };
  auto edge = [&](int q) { return edge_of(f, q); };
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f;
  const bool by_count = k > 0 && k < V, by_mass = p < 1.f;
  float pmin = a.min_p ? a.min_p[r] : 0.f;
  pmin = pmin > 1.f ? 1.f : pmin;
  // the lowest logit that has a weight: below it (and NaN) nothing matters
  const float cut = of_key(lowest_key(kmax, gmax - 22.180709f / f.inv, [&](float x) { return Row::w(f.e(x)) > 0; }));
  const uint32_t key_pmin = pmin > 0.f ? lowest_key(kmax, gmax + logf(pmin) / f.inv, [&](float x) { return f.e(x) >= pmin; }) : 0;
  u64 thr = 0;  // rank word of the last element that is kept

  if (by_count && k <= FAST_K) {
    if (m0 >= cut) atomicAdd(&s.hc[bin(m0) / BINS], 1u);
    if (m1 >= cut) atomicAdd(&s.hc[bin(m1) / BINS], 1u);
    __syncthreads();
    // The row's k largest elements lie in the bins up to the one that holds this
    // CTA's k-th largest thread maximum, or up to the last of those that hold the
    // CTAs' k / C-th: both from all CTAs, the best of them bounds the row.
    {
      const u64 part = (k + C - 1) / C;
      u64 all, v[BINS / NT], own = 0;
#pragma unroll
      for (int i = 0; i < BINS / NT; ++i) own += v[i] = s.hc[tid * (BINS / NT) + i];
      if (tid == 0) s.bounds[0] = s.bounds[1] = BINS;
      u64 before = scan(s, own, &all);
#pragma unroll
      for (int i = 0; i < BINS / NT; ++i) {
        if (before < (u64)k && (u64)k <= before + v[i]) s.bounds[0] = tid * (BINS / NT) + i;
        if (before < part && part <= before + v[i]) s.bounds[1] = tid * (BINS / NT) + i;
        before += v[i];
      }
      __syncthreads();
      if (tid < C) {
        cluster.map_shared_rank(&s.counts[0][0], tid)[rank] = s.bounds[0];
        cluster.map_shared_rank(&s.counts[1][0], tid)[rank] = s.bounds[1];
      }
    }
    cluster.sync();
    int b = BINS, parts = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      b = min(b, s.counts[0][c]);
      parts = max(parts, s.counts[1][c]);
    }
    b = min(b, parts);
    const float cut_k = b < BINS ? fmaxf(cut, edge(BINS * b + BINS - 1)) : cut;
    int mine = 0;
    x.each(cut_k, [&](float y, int i) {
      ++mine;
      const int at = atomicAdd(cluster.map_shared_rank(&s.n_list, 0), 1);
      if (at < CAP) cluster.map_shared_rank(s.list, 0)[at] = rank_word(key_of(y), i);
    });
    mine = reduce(mine, [](int x, int y) { return x + y; }, reinterpret_cast<int *>(s.red));
    if (tid < C) cluster.map_shared_rank(s.found, tid)[rank] = mine;
    cluster.sync();
    int sum = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) sum += s.found[c];
    if (sum <= CAP) {
      if (rank == 0) draw_sorted(s, a, r, f, sum, k, p, key_pmin);
      return;
    }
    if (tid == 0) s.n_list = 0;
    for (int i = tid; i < BINS; i += NT) s.hc[i] = 0;
    __syncthreads();
  }

  // top-k, then top-p
  if (by_count || by_mass) {
    // fine bins `base` .. of 2^shift each: counts and weights of the row's elements in 512 of them, to every CTA
    auto histogram = [&](float from, float end, int base, int shift) {
      x.between(from, end, [&](const float (&y)[VEC], int) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          if (!(y[i] >= from) || y[i] >= end) continue;
          const u64 w = f.weight(y[i]);
          const int b = (bin(y[i]) - base) >> shift;
          if (by_count) atomicAdd(&s.hc[b], 1u);
          atomicAdd(&s.hl[b], (uint32_t)w & 0xffffu);
          atomicAdd(&s.hh[b], (uint32_t)(w >> 16));
        }
      });
      cluster.sync();
      for (int b = rank * (BINS / C) + tid; b < (rank + 1) * (BINS / C); b += NT) {
        uint32_t c = 0;
        u64 w = 0;
#pragma unroll
        for (int o = 0; o < C; ++o) {
          c += cluster.map_shared_rank(s.hc, o)[b];
          w += cluster.map_shared_rank(s.hl, o)[b] + ((u64)cluster.map_shared_rank(s.hh, o)[b] << 16);
        }
#pragma unroll
        for (int o = 0; o < C; ++o) {
          cluster.map_shared_rank(s.row_c, o)[b] = c;
          cluster.map_shared_rank(s.row_w, o)[b] = w;
        }
      }
      cluster.sync();
    };
    auto weight_before = [&](int n) {  // of the first n bins
      u64 v = 0;
      for (int i = tid; i < n; i += NT) v += s.row_w[i];
      return block_total(s, v);
    };
    const float none = __uint_as_float(0x7fc00000u);  // NaN: no logit is at or above it
    histogram(cut, none, 0, 9);
    u64 W = weight_before(BINS);  // weight that top-p divides
    int fine = -1;  // the bin that has been looked at closer
#pragma unroll 1
    for (int round = 0; round < 2; ++round) {
      const bool mass = round;
      if (!(mass ? by_mass : by_count)) continue;
      const u64 target = mass ? share_of(p, W) : (u64)k;
      if (fine >= 0) {  // top-k looked closer into a bin: the whole range again
        for (int i = tid; i < BINS; i += NT) s.hc[i] = s.hl[i] = s.hh[i] = 0;
        __syncthreads();
        histogram(cut, none, 0, 9);
        fine = -1;
      }
      float from = cut, end = none;
      u64 before = 0, above_w = 0;  // of what lies above the range: the round's measure, and the weight
      int base = 0, shift = 9;
      int n = 0;
      while (true) {
        const int b = crossing<BINS>(s, target - before, [&](int i) { return mass ? s.row_w[i] : (u64)s.row_c[i]; });
        if (b < 0) break;  // fewer elements have a weight (a rounding at most, for a weight)
        before += s.out[0];
        above_w += weight_before(b);
        const int q = base + (b << shift);
        from = fmaxf(from, edge(q + (1 << shift) - 1));
        const float up = edge(q - 1);
        end = b ? up : end;
        // the bin's elements, to every CTA (each has them in an order of its own)
        x.between(from, end, [&](const float (&y)[VEC], int first) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            if (!(y[i] >= from) || y[i] >= end) continue;
            const int at = atomicAdd(&s.n_own, 1);
            if (at < OWN) s.own[at] = rank_word(key_of(y[i]), first + i);
          }
        });
        __syncthreads();
        const int mine = s.n_own;
        if (tid < C) cluster.map_shared_rank(&s.counts[shift ? 0 : 1][0], tid)[rank] = mine;
        cluster.sync();
        int first = 0;
        bool fits = true;
        n = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int m = s.counts[shift ? 0 : 1][c];
          if (c == rank) first = n;
          fits &= m <= OWN;
          n += m;
        }
        fits &= n <= CAP;
        if (fits) {
          for (int i = tid; i < C * mine; i += NT) {
            const int to = i / mine, j = i - to * mine;
            cluster.map_shared_rank(s.list, to)[first + j] = s.own[j];
          }
          cluster.sync();
          break;
        }
        n = 0;
        if (shift == 0) break;
        if (tid == 0) s.n_own = 0;
        for (int i = tid; i < BINS; i += NT) s.hc[i] = s.hl[i] = s.hh[i] = 0;
        __syncthreads();
        base = fine = q;
        shift = 0;
        histogram(from, end, base, 0);
      }
      const bool ok = n > 0;
      u64 found = 0, found_w = 0;
      if (ok) {
        // narrow the list's range of rank words until few are left
        u64 lo = 0, hi = ~0ull >> 1;
        int in = n;
        while (in > FEW) {
          u64 mn = ~0ull, mx = 0;
          for (int i = tid; i < n; i += NT) {
            const u64 word = s.list[i];
            if (word < lo || word > hi) continue;
            mn = min(mn, word);
            mx = max(mx, word);
          }
          lo = reduce(mn, [](u64 x, u64 y) { return x < y ? x : y; }, s.red);
          hi = reduce(mx, [](u64 x, u64 y) { return x > y ? x : y; }, s.red);
          const int down = max(0, 64 - __clzll(hi - lo) - 3);
          u64 m[8], c[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) m[j] = c[j] = 0;
          for (int i = tid; i < n; i += NT) {
            const u64 word = s.list[i];
            if (word < lo || word > hi) continue;
            const u64 w = f.weight(of_key((uint32_t)(word >> IDX_BITS)));
            const int g = (int)((hi - word) >> down);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              m[j] += g == j ? w : 0;
              c[j] += g == j;
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int w = 16; w; w >>= 1) {
              m[j] += __shfl_xor_sync(0xffffffffu, m[j], w);
              c[j] += __shfl_xor_sync(0xffffffffu, c[j], w);
            }
            if (lane == 0) {
              s.part_red[warp][j] = m[j];
              s.part_red[warp][8 + j] = c[j];
            }
          }
          __syncthreads();
          int g = 0;
          for (; g < 8; ++g) {
            u64 gm = 0, gc = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
              gm += s.part_red[w][g];
              gc += s.part_red[w][8 + g];
            }
            if (before + (mass ? gm : gc) >= target || g == 7) {
              in = (int)gc;
              break;
            }
            before += mass ? gm : gc;
            above_w += gm;
          }
          __syncthreads();
          hi -= (u64)g << down;
          const u64 size = ((u64)1 << down) - 1;
          lo = hi - lo > size ? hi - size : lo;
        }
        if (tid == 0) {
          s.n_few = 0;
          s.out[0] = 0;
        }
        __syncthreads();
        for (int i = tid; i < n; i += NT) {
          const u64 word = s.list[i];
          if (word < lo || word > hi) continue;
          const int at = atomicAdd(&s.n_few, 1);
          s.few[at] = word;
        }
        __syncthreads();
        // largest first, the element at which the running count or weight reaches the target
        u64 me = tid < in ? s.few[tid] : 0;
        sort_down_few(s.few, me, in);
        const u64 w = me ? f.weight(of_key((uint32_t)(me >> IDX_BITS))) : 0;
        u64 all;
        const u64 m = scan(s, w, &all), ex = before + (mass ? m : (u64)tid), own = mass ? w : 1;
        if (me && ex < target && target <= ex + own) {
          s.out[0] = me;
          s.out[1] = above_w + m + w;
        }
        __syncthreads();
        found = s.out[0];
        found_w = s.out[1];
      }
      if (!found) found = find_slowly<T, C>(s, x, f, cut, !mass, target, thr, &found_w);
      thr = max(thr, found);
      W = found_w;
      if (round == 0 && by_mass) {  // the list is used again
        cluster.sync();
        if (tid == 0) s.n_own = 0;
        __syncthreads();
      }
    }
  }

  // the kept weight of each warp, to everyone
  const bool filtered = thr || key_pmin;
  const float from = fmaxf(fmaxf(cut, thr ? of_key((uint32_t)(thr >> IDX_BITS)) : -INFINITY), key_pmin ? of_key(key_pmin) : -INFINITY);
  const float tie = thr ? of_key((uint32_t)(thr >> IDX_BITS)) : -INFINITY;
  const int tie_idx = (int)(MAX_VOCAB - 1 - (thr & (MAX_VOCAB - 1)));
  auto kept = [&](float y, int i) -> u64 {
    const u64 w = f.weight(y);
    return y >= from && !(y == tie && i > tie_idx) ? w : 0;
  };
  u64 sum_kept = 0;
  auto add_kept = [&](const float (&y)[VEC], int first) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum_kept += kept(y[i], first + i);
  };
  if (filtered) {
    x.template vectors<true>(from, add_kept);
  } else {
    x.template vectors<false>(from, [&](const float (&y)[VEC], int) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum_kept += f.weight(y[i]);
    });
  }
#pragma unroll
  for (int w = 16; w; w >>= 1) sum_kept += __shfl_xor_sync(0xffffffffu, sum_kept, w);
  if (lane < C) cluster.map_shared_rank(&s.warp_sums[0][0], lane)[rank * NW + warp] = sum_kept;
  cluster.sync();

  // the warp in which the running sum passes the place
  static_assert(C * NW <= 64, "two sums a lane");
  u64 total, before, mine = (&s.warp_sums[0][0])[rank * NW + warp];
  {
    const bool in = 2 * lane < C * NW;
    const u64 s0 = in ? (&s.warp_sums[0][0])[2 * lane] : 0, s1 = in ? (&s.warp_sums[0][0])[2 * lane + 1] : 0;
    u64 up = s0 + s1;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, up, w);
      if (lane >= w) up += y;
    }
    total = __shfl_sync(0xffffffffu, up, 31);
    const int me = rank * NW + warp;
    before = __shfl_sync(0xffffffffu, up - (me & 1 ? s1 : s0 + s1), me / 2);
  }
  const u64 at = place(a.u[r], total);
  if (before <= at && at < before + mine) {
    for (int v = x.v0; v < x.v1; v += 32) {
      const bool in = v + lane < x.v1;
      const uint4 q = in ? x.xv[v + lane] : make_uint4(0, 0, 0, 0);
      const int first = i0 + (v + lane) * VEC;
      u64 own = 0;
      if (in) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) own += kept(X::get(q, j), first + j);
      }
      u64 sum = own;
#pragma unroll
      for (int w = 1; w < 32; w <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, sum, w);
        if (lane >= w) sum += y;
      }
      const uint32_t over = __ballot_sync(0xffffffffu, before + sum > at);
      if (over) {
        if (lane == __ffs(over) - 1) {
          u64 c = before + sum - own;
          int j = 0;
          for (; j < VEC - 1; ++j) {
            c += kept(X::get(q, j), first + j);
            if (c > at) break;
          }
          a.tokens[r] = first + j;
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
}

template <class T, int C>
int launch_cluster(const Args &a, int slice, cudaStream_t st, int device) {
  const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + (size_t)slice * sizeof(T);
  static ContextOnce attr;
  if (int s = attr.run(device, []() -> int {
        NKB_CUDA_TRY(cudaFuncSetAttribute(cluster_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        return NKB_OK;
      }))
    return s;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * C));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  NKB_CUDA_TRY(cudaLaunchKernelEx(&cfg, cluster_kernel<T, C>, a, slice));
  return launch_status("sample_tokens");
}

// elements of a CTA of c, and its shared memory
int slice_of(const Args &a, int c) { return (int)(((a.vocab + c - 1) / c + 7) / 8 * 8); }
size_t smem_of(const Args &a, int c) { return (sizeof(Shared) + 15) / 16 * 16 + (size_t)slice_of(a, c) * dtype_size((int)a.dtype); }

// CTAs per row; 0: the row does not fit a cluster.  Eight for few rows; where that
// makes more than two CTAs per SM, half as many while two still fit an SM: CTAs
// that wait for a place cost more than longer slices.  Measured with top-p 0.95,
// bf16, us with 8 / 4 / 2 / 1 CTAs per row: 8 rows of 32000 fp32 21 / 25 / 34 / 55,
// 32 x 32000 26 / 23 / 33 / 48, 128 x 32000 81 / 51 / 40 / 50, 512 x 32000 288 /
// 142 / 111 / 109, 128 x 151936 173 / 142 / 198 / -; with top-k 50 300 x 2000 55 /
// 33 / 23 / 12.
int cluster_of(const Args &a, int device) {
  if (slice_of(a, MAX_C) > MAX_SLICE || smem_of(a, MAX_C) > 227 * 1024) return 0;
  int c = MAX_C;
  while (c > 1 && a.rows * c > 2 * num_sms(device) && smem_of(a, c / 2) <= 113 * 1024) c /= 2;
  return c;
}

template <class T>
int launch_rows(const Args &a, int c, cudaStream_t st, int device) {
  if (c == 1) return launch_cluster<T, 1>(a, slice_of(a, c), st, device);
  if (c == 2) return launch_cluster<T, 2>(a, slice_of(a, c), st, device);
  if (c == 4) return launch_cluster<T, 4>(a, slice_of(a, c), st, device);
  return launch_cluster<T, 8>(a, slice_of(a, c), st, device);
}

// ---- rows of any length ------------------------------------------------------
// One block per row, the logits read from memory for every step: for rows that
// are too long for a cluster's shared memory.  The threshold is found bit by
// bit; `quota` of the elements equal to it are kept, in index order.
constexpr int THREADS = 1024;

template <class V, class Op>
__device__ V block_reduce(V v, Op op, V *shared) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int w = 16; w; w >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, w));
  __syncthreads();  // earlier readers of `shared` are done
  if (lane == 0) shared[warp] = v;
  __syncthreads();
  v = shared[lane];  // THREADS / 32 == 32 warps
#pragma unroll
  for (int w = 16; w; w >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, w));
  return v;
}

__global__ void __launch_bounds__(THREADS) long_row_kernel(const __grid_constant__ Args a) {
  __shared__ u64 red[32];
  __shared__ u64 warp_sum[32];
  __shared__ int found;
  const int64_t r = blockIdx.x;
  const int V = (int)a.vocab, dt = (int)a.dtype, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const char *row = static_cast<const char *>(a.logits) + r * a.row_stride * (dt == NKB_F32 ? 4 : 2);
  auto add = [](u64 x, u64 y) { return x + y; };
  auto lower = [](u64 x, u64 y) { return x < y ? x : y; };
  auto higher = [](u64 x, u64 y) { return x > y ? x : y; };

  // largest key, and the lowest index that has it
  u64 best = 0;
  for (int i = tid; i < V; i += THREADS) {
    const u64 v = ((u64)key_of(load_x(row, i, dt)) << 32) | (uint32_t)~i;
    best = best > v ? best : v;
  }
  best = block_reduce(best, higher, red);
  const uint32_t kmax = (uint32_t)(best >> 32);
  const int first = (int)~(uint32_t)best;
  if (kmax <= KEY_NEG_INF) {
    if (tid == 0) a.tokens[r] = -1;
    return;
  }
  const float temp = a.temperature ? a.temperature[r] : 1.f;
  if (!(temp > 0.f)) {
    if (tid == 0) a.tokens[r] = first;
    return;
  }
  const Row f(of_key(kmax), temp);

  uint32_t tau = 0;    // threshold key
  u64 quota = ~0ull;   // elements equal to tau that are kept
  const int k = a.top_k ? a.top_k[r] : 0;
  if (k > 0 && k < V) {
    // the largest key that at least k elements reach, bit by bit from the top
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = tau | (1u << bit);
      u64 n = 0;
      for (int i = tid; i < V; i += THREADS) n += key_of(load_x(row, i, dt)) >= t;
      if (block_reduce(n, add, red) >= (u64)k) tau = t;
    }
    u64 n = 0;
    for (int i = tid; i < V; i += THREADS) n += key_of(load_x(row, i, dt)) > tau;
    quota = (u64)k - block_reduce(n, add, red);
  }
  const float p = a.top_p ? a.top_p[r] : 1.f;
  if (p < 1.f) {
    // weight of the elements with key >= t, at most `quota` of those equal to tau
    auto mass = [&](uint32_t t) {
      u64 s = 0, ties = 0, wt = 0;
      for (int i = tid; i < V; i += THREADS) {
        const float x = load_x(row, i, dt);
        const uint32_t key = key_of(x);
        if (key > tau && key >= t) s += Row::w(f.e(x));
        if (key == tau && key >= t) {
          ++ties;
          wt = Row::w(f.e(x));
        }
      }
      s = block_reduce(s, add, red);
      ties = block_reduce(ties, add, red);
      wt = block_reduce(wt, higher, red);
      return s + (ties < quota ? ties : quota) * wt;
    };
    const u64 W = mass(0);
    const u64 T = share_of(p, W);
    uint32_t t = 0;
    for (int bit = 31; bit >= 0; --bit)
      if (mass(t | (1u << bit)) >= T) t |= 1u << bit;
    const u64 above = t == 0xffffffffu ? 0 : mass(t + 1);
    const u64 wt = Row::w(f.e(of_key(t)));
    const u64 q = wt ? (T - above + wt - 1) / wt : ~0ull;
    quota = t == tau ? (q < quota ? q : quota) : q;
    tau = t;
  }
  float pmin = a.min_p ? a.min_p[r] : 0.f;
  pmin = pmin > 1.f ? 1.f : pmin;

  // kept weight of each warp's contiguous part: sum above tau and ties
  const int part = ((V + 31) / 32 + 31) / 32 * 32, i0 = warp * part, i1 = min(i0 + part, V);
  const float xt = of_key(tau);
  const bool tie_in = tau > KEY_NEG_INF && !(f.e(xt) < pmin);
  const u64 wt = tie_in ? Row::w(f.e(xt)) : 0;
  u64 s = 0, ties = 0;
  for (int i = i0 + lane; i < i1; i += 32) {
    const float x = load_x(row, i, dt), e = f.e(x);
    const uint32_t key = key_of(x);
    if (key > tau && !(e < pmin)) s += Row::w(e);
    if (key == tau) ++ties;
  }
#pragma unroll
  for (int w = 16; w; w >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, w);
    ties += __shfl_xor_sync(0xffffffffu, ties, w);
  }
  __syncthreads();
  if (lane == 0) {
    warp_sum[warp] = s;
    red[warp] = ties;
  }
  if (tid == 0) found = first;
  __syncthreads();
  u64 before = 0, ties_before = 0, S = 0, N = 0;
  for (int w = 0; w < 32; ++w) {
    if (w == warp) {
      before = S;
      ties_before = N;
    }
    S += warp_sum[w];
    N += red[w];
  }
  auto upto = [&](u64 sum, u64 n) { return sum + (n < quota ? n : quota) * wt; };
  const u64 total = upto(S, N);
  const u64 at = place(a.u[r], total);
  if (upto(before, ties_before) <= at && at < upto(before + s, ties_before + ties)) {
    for (int base = i0; base < i1; base += 32) {
      const int i = base + lane;
      u64 ws = 0, nt = 0;
      if (i < i1) {
        const float x = load_x(row, i, dt), e = f.e(x);
        const uint32_t key = key_of(x);
        if (key > tau && !(e < pmin)) ws = Row::w(e);
        nt = key == tau;
      }
#pragma unroll
      for (int w = 1; w < 32; w <<= 1) {
        const u64 p1 = __shfl_up_sync(0xffffffffu, ws, w), p2 = __shfl_up_sync(0xffffffffu, nt, w);
        if (lane >= w) {
          ws += p1;
          nt += p2;
        }
      }
      const uint32_t over = __ballot_sync(0xffffffffu, upto(before + ws, ties_before + nt) > at);
      if (over) {
        if (lane == 0) found = base + __ffs(over) - 1;
        break;
      }
      before += __shfl_sync(0xffffffffu, ws, 31);
      ties_before += __shfl_sync(0xffffffffu, nt, 31);
    }
  }
  __syncthreads();
  if (tid == 0) a.tokens[r] = found;
}


int check_args(const Args &a) {
  auto bad = [](const char *m) { return fail(NKB_ERR_INVALID, std::string("sample_tokens: ") + m); };
  if (a.rows < 0 || a.rows > INT32_MAX / MAX_C || a.vocab < 1) return bad("rows or vocab out of range");
  if (a.dtype != NKB_F32 && a.dtype != NKB_BF16 && a.dtype != NKB_F16)
    return fail(NKB_ERR_UNSUPPORTED, "sample_tokens: logits must be float32, bfloat16 or float16");
  if (a.vocab > MAX_VOCAB) return fail(NKB_ERR_UNSUPPORTED, "sample_tokens: more than 2^21 entries");
  if (a.rows && (!a.logits || !a.u || !a.tokens)) return bad("NULL array");
  if (a.rows > 1 && a.row_stride < a.vocab) return bad("rows overlap");
  return NKB_OK;
}

int run(const Args &a, cudaStream_t st, int device) {
  if (int s = check_args(a)) return s;
  if (a.rows == 0) return NKB_OK;
  if (const int c = cluster_of(a, device)) {
    if (a.dtype == NKB_F32) return launch_rows<float>(a, c, st, device);
    if (a.dtype == NKB_BF16) return launch_rows<__nv_bfloat16>(a, c, st, device);
    return launch_rows<__half>(a, c, st, device);
  }
  long_row_kernel<<<(unsigned)a.rows, THREADS, 0, st>>>(a);
  return launch_status("sample_tokens");
}

// "sample_tokens": the pointers of nkb_sample_args that are given; ints a mask of
// them and the struct's integers
int check(const Step &s) {
  Args a;
  if (int e = paged::step_args(s, nullptr, 7, 4, "sample_tokens", &a)) return e;
  return check_args(a);
}
int launch(const LaunchArgs &l) {
  Args a;
  if (int e = paged::step_args(*l.step, l.ptrs, 7, 4, "sample_tokens", &a)) return e;
  return run(a, l.stream, l.device);
}

}  // namespace sample

NKB_REGISTER_KERNEL("sample_tokens", sample::launch, sample::check);

}  // namespace nkb

extern "C" int nkb_sample_tokens(const nkb_sample_args *args, void *stream) {
  if (!args) return nkb::fail(NKB_ERR_INVALID, "args is NULL");
  int dev = 0;
  cudaGetDevice(&dev);
  return nkb::sample::run(*args, static_cast<cudaStream_t>(stream), dev);
}
