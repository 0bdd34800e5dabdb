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
// A cluster of 8 CTAs holds a row in its shared memory: the logits are read from
// memory once.  What bounds the kernel is then the instructions per element and
// the cluster's meetings, so that elements which cannot matter are dropped by
// one comparison with a cut: the lowest logit with a nonzero weight, and for
// top-k a bound from the threads' own maxima.
//   1  logits to shared memory, each thread's maxima; the row's maximum
//   2  top-k of up to FAST_K: what passes the bound (some 8 k elements) goes to
//      one CTA, which sorts it and does the rest alone; otherwise
//   3  top-k / top-p: histogram of counts and weights over bins linear in
//      (max - x) / temperature; summed over the cluster, every CTA gets it
//   4  the elements of the bin that the threshold falls in go to every CTA,
//      which finds the threshold among them (narrowing by rank word)
//   5  kept weight per warp, contiguous in the row; the warp in which the
//      running sum passes u times the total walks its part
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

struct Row {
  float max, inv;  // largest logit, 1 / temperature
  __device__ __forceinline__ float t(float x) const { return __fmul_rn(__fsub_rn(x, max), inv); }
  __device__ __forceinline__ float e(float x) const { return x == max ? 1.f : x == -INFINITY ? 0.f : expf(t(x)); }
  // floor(2^32 e) for e in [0, 1]: the significand, moved
  static __device__ __forceinline__ u64 w(float e) {
    const uint32_t b = __float_as_uint(e);
    const int down = 126 - (int)(b >> 23);
    if (down < 0) return 1ull << 32;  // e = 1
    return down > 31 ? 0 : (((b & 0x7fffffu) | 0x800000u) << 8) >> down;
  }
};

// ---- rows in a cluster's shared memory -------------------------------------
constexpr int NT = 512, NW = NT / 32;
constexpr int NB = 1024;    // bins
constexpr int CAP = 1024;   // elements of a bin that a CTA takes
constexpr int FEW = 96;     // elements that are ranked one against another
constexpr int C = 8;        // CTAs of a cluster
constexpr int FAST_K = 100; // top-k that one CTA sorts: C * FAST_K candidates are expected, CAP fit
constexpr int MAX_SLICE = 65528;  // weights' 16-bit halves sum to less than 2^32
constexpr float SPAN = 22.25f;    // e^-SPAN < 2^-32

struct Shared {
  u64 list[2][CAP], lw[2][CAP];  // rank words and weights of the threshold bin: top-k's, top-p's
  u64 gm[NB];                    // weights per bin, whole row
  u64 sums[C], red[NW], red2[NW], few[FEW], few_w[FEW];
  uint32_t hc[NB], hl[NB], hh[NB];  // this CTA's bins: counts, low and high halves of the weights
  uint32_t gc[NB];                  // counts per bin, whole row
  uint32_t nc[NB], nl[NB], nh[NB];  // narrowing
  float maxima[C];
  int counts[C], n_fast;
  u64 out_a, out_b, out_c;
  int n_list, bin;
};

template <class V, class Op>
__device__ V reduce(V v, Op op, V *shared) {  // over the block, to every thread
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

// Lowest key in (-inf, inf] that `yes` holds for, where it holds for `top` and
// for every key above one it holds for: by one warp, first the 32 keys around a
// guess, then 32 pivots at a time.
template <class Yes>
__device__ uint32_t lowest_key(uint32_t top, float guess, Yes yes) {
  uint32_t lo = KEY_NEG_INF, hi = top;  // not at lo, at hi
  const int lane = threadIdx.x & 31;
  {
    const uint32_t g = key_of(guess);
    const uint32_t base = g > KEY_NEG_INF + 16 && g < top ? g - 16 : KEY_NEG_INF;
    const uint32_t at = min(base + 1 + lane, hi);
    const uint32_t m = __ballot_sync(0xffffffffu, yes(of_key(at)));
    const int f = __ffs(m) - 1;
    if (f > 0) return min(base + 1 + f, hi);
    if (f == 0) hi = min(base + 1, hi);
    else lo = base + 32;
  }
  while (hi - lo > 1) {
    const uint32_t step = (hi - lo - 1) / 32 + 1;
    const uint32_t off = step * (lane + 1), at = off < hi - lo ? lo + off : hi;
    const uint32_t m = __ballot_sync(0xffffffffu, yes(of_key(at)));
    const int f = __ffs(m) - 1;  // the last pivot is hi or above it
    const uint32_t up = step * (f + 1);
    hi = up < hi - lo ? lo + up : hi;
    lo += step * f;
  }
  return hi;
}

// First bin, from bin 0, in which the running sum of get(bin) reaches `target`
// (the last one if none does): its index and the sum before it, to every thread.
template <int N, class Get>
__device__ int crossing(Shared &s, u64 target, Get get, u64 *before) {
  constexpr int PER = N / NT;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  u64 v[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) sum += v[i] = get(tid * PER + i);
  u64 x = sum;
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, x, w);
    if (lane >= w) x += y;
  }
  __syncthreads();
  if (lane == 31) s.red[warp] = x;
  if (tid == 0) s.bin = N;
  __syncthreads();
  u64 at = x - sum;
  for (int w = 0; w < warp; ++w) at += s.red[w];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (at < target && target <= at + v[i]) {
      s.bin = tid * PER + i;
      s.out_a = at;
    }
    at += v[i];
  }
  __syncthreads();
  *before = s.out_a;
  return s.bin;
}

// The rest of a row whose n candidates (rank words, at most CAP) hold its k
// largest elements, by one CTA.
__device__ void draw_sorted(Shared &s, const Args &a, int64_t r, const Row &f, int n, int k, float p, uint32_t key_pmin) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  u64 *list = s.list[0];
  int N = 64;
  while (N < n) N *= 2;
  for (int i = n + tid; i < N; i += NT) list[i] = 0;
  __syncthreads();
  // bitonic, largest first; a warp keeps the 64 elements of its short strides to itself
  for (int size = 2; size <= N; size *= 2)
    for (int stride = size / 2; stride; stride /= 2) {
      if (tid < N / 2) {
        const int i = 2 * tid - (tid & (stride - 1)), j = i + stride;
        const u64 x = list[i], y = list[j];
        if ((x < y) == ((i & size) == 0)) {
          list[i] = y;
          list[j] = x;
        }
      }
      // the next stride's elements are this warp's own while it is at most 32
      if (stride > 1 && stride <= 32) __syncwarp();
      else __syncthreads();
    }
  const int m = min(k, n);
  static_assert(FAST_K <= 128, "four warps hold the k largest");
  u64 w = 0, sum = 0;
  uint32_t key = 0;
  if (tid < 128) {
    if (tid < m) {
      key = (uint32_t)(list[tid] >> IDX_BITS);
      w = Row::w(f.e(of_key(key)));
    }
    sum = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += y;
    }
    if (lane == 31) s.red[warp] = sum;
  }
  __syncthreads();
  if (tid < 128) {
    for (int i = 0; i < warp; ++i) sum += s.red[i];
    const u64 W = s.red[0] + s.red[1] + s.red[2] + s.red[3];
    const double want = (double)p * (double)W;
    const u64 T = p < 1.f ? (want >= 1.0 ? (u64)want : 1) : ~0ull;
    const bool keep = tid < m && sum - w < T && key >= key_pmin;
    s.lw[0][tid] = keep ? w : 0;
  }
  __syncthreads();
  if (tid < 128) {
    const u64 own = s.lw[0][tid];
    u64 total = 0, upto = 0;  // of all, and of those up to this one in index order
    for (int i = 0; i < m; ++i) {
      const u64 x = s.lw[0][i];
      total += x;
      if (tid < m && (list[i] & (MAX_VOCAB - 1)) >= (list[tid] & (MAX_VOCAB - 1))) upto += x;
    }
    const float u = a.u[r];
    u64 at = (u64)((double)(u > 0.f ? u : 0.f) * (double)total);
    at = at < total ? at : total - 1;
    if (own && upto > at && upto - own <= at) a.tokens[r] = (int)(MAX_VOCAB - 1 - (list[tid] & (MAX_VOCAB - 1)));
  }
}

template <class T>
__global__ void __launch_bounds__(NT, 2) cluster_kernel(const __grid_constant__ Args a, int slice) {
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t smem[];
  Shared &s = *reinterpret_cast<Shared *>(smem);
  T *xs = reinterpret_cast<T *>(smem + (sizeof(Shared) + 15) / 16 * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x / C;
  const int V = (int)a.vocab, i0 = rank * slice, n = max(0, min(slice, V - i0));
  const T *row = static_cast<const T *>(a.logits) + r * a.row_stride + i0;
  // vectors of this warp: contiguous, [v0, v1)
  const int nv = (n + VEC - 1) / VEC, per = (nv + NW - 1) / NW, v0 = min(nv, warp * per), v1 = min(nv, v0 + per);
  auto get = [](const uint4 &q, int j) -> float {
    const uint32_t w = (&q.x)[j / (VEC / 4)];
    float x;
    if constexpr (sizeof(T) == 4) x = __uint_as_float(w);
    else if constexpr (std::is_same<T, __half>::value) x = __half2float(__ushort_as_half((unsigned short)(j & 1 ? w >> 16 : w)));
    else x = __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
    return x + 0.f;
  };
  const uint4 *xv = reinterpret_cast<const uint4 *>(xs);

  // 1  logits to shared memory; the tail of the last vector is -inf
  float m0 = -INFINITY, m1 = -INFINITY;  // this thread's maxima: even and odd steps
  if ((reinterpret_cast<uintptr_t>(row) & 15) == 0) {
    const uint4 *src = reinterpret_cast<const uint4 *>(row);
    const int full = n / VEC;
#pragma unroll 4
    for (int v = tid; v < full; v += NT) reinterpret_cast<uint4 *>(xs)[v] = __ldcs(src + v);
    for (int i = full * VEC + tid; i < nv * VEC; i += NT) xs[i] = i < n ? row[i] : (T)(-INFINITY);
  } else {
#pragma unroll 4
    for (int i = tid; i < nv * VEC; i += NT) xs[i] = i < n ? row[i] : (T)(-INFINITY);
  }
  __syncthreads();
  for (int v = v0 + lane, odd = 0; v < v1; v += 32, odd ^= 1) {
    const uint4 q = xv[v];
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < VEC; ++j) m = fmaxf(m, get(q, j));  // NaN is passed over
    if (odd) m1 = fmaxf(m1, m);
    else m0 = fmaxf(m0, m);
  }
  {
    const float m = reduce(fmaxf(m0, m1), [](float x, float y) { return fmaxf(x, y); }, reinterpret_cast<float *>(s.red));
    if (tid < C) cluster.map_shared_rank(s.maxima, tid)[rank] = m;
  }
  if (tid == 0) s.n_fast = 0;
  cluster.sync();
  float gmax = -INFINITY;
  int owner = 0;  // lowest rank that has the maximum
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
  auto add = [](u64 x, u64 y) { return x + y; };
  auto low = [](u64 x, u64 y) { return x < y ? x : y; };
  auto high = [](u64 x, u64 y) { return x > y ? x : y; };
  if (!(temp > 0.f)) {
    if (rank != owner) return;
    u64 first = V;
    for (int v = v0 + lane; v < v1; v += 32) {
      const uint4 q = xv[v];
      for (int j = VEC - 1; j >= 0; --j)
        if (get(q, j) == gmax) first = min(first, (u64)(i0 + v * VEC + j));
    }
    first = reduce(first, low, s.red);
    if (tid == 0) a.tokens[r] = (int)first;
    return;
  }

  const Row f{gmax, 1.f / temp};
  const uint32_t kmax = key_of(gmax);
  auto bin_of = [&](float x) { return min(NB - 1, (int)__fmul_rn(f.t(x), -(float)NB / SPAN)); };
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f;
  const bool by_count = k > 0 && k < V, by_mass = p < 1.f;
  float pmin = a.min_p ? a.min_p[r] : 0.f;
  pmin = pmin > 1.f ? 1.f : pmin;
  // the lowest logit that has a weight: below it (and NaN) nothing matters
  float cut = of_key(lowest_key(kmax, gmax - 22.180709f * temp, [&](float x) { return Row::w(f.e(x)) > 0; }));
  // lowest logit of the bins up to b
  auto bin_end = [&](int b) {
    return lowest_key(kmax, gmax - (float)(b + 1) * (SPAN / NB) * temp, [&](float x) { return bin_of(x) <= b; });
  };
  const uint32_t key_pmin = pmin > 0.f ? lowest_key(kmax, gmax + logf(pmin) * temp, [&](float x) { return f.e(x) >= pmin; }) : 0;
  u64 thr = 0;  // rank word of the last kept element

  if (by_count || by_mass) {
    for (int i = tid; i < NB; i += NT) s.hc[i] = s.hl[i] = s.hh[i] = 0;
    __syncthreads();
    float cut_k = cut;
    if (by_count && k <= 2 * NT) {
      // k of this CTA's thread maxima lie in the bins up to b: so do the row's k largest
      if (m0 >= cut) atomicAdd(&s.hc[bin_of(m0)], 1u);
      if (m1 >= cut) atomicAdd(&s.hc[bin_of(m1)], 1u);
      __syncthreads();
      u64 before;
      const int b = crossing<NB>(s, (u64)k, [&](int i) { return (u64)s.hc[i]; }, &before);
      if (b < NB) cut_k = fmaxf(cut, of_key(bin_end(b)));
      if (k <= FAST_K) {
        // 2  candidates to rank 0; how many there are, to everyone
        int mine = 0;
        for (int v = v0 + lane; v < v1; v += 32) {
          const uint4 q = xv[v];
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float x = get(q, j);
            if (x >= cut_k) {
              ++mine;
              const int at = atomicAdd(cluster.map_shared_rank(&s.n_fast, 0), 1);
              if (at < CAP) cluster.map_shared_rank(s.list[0], 0)[at] = rank_word(key_of(x), i0 + v * VEC + j);
            }
          }
        }
        mine = reduce(mine, [](int x, int y) { return x + y; }, reinterpret_cast<int *>(s.red));
        if (tid < C) cluster.map_shared_rank(s.counts, tid)[rank] = mine;
        cluster.sync();
        int all = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) all += s.counts[c];
        if (all <= CAP) {
          if (rank == 0) draw_sorted(s, a, r, f, all, k, p, key_pmin);
          return;
        }
      }
      for (int i = tid; i < NB; i += NT) s.hc[i] = 0;
      __syncthreads();
    }
    // 3  histogram
    for (int v = v0 + lane; v < v1; v += 32) {
      const uint4 q = xv[v];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float x = get(q, j);
        if (x >= cut_k) {
          const u64 full = Row::w(f.e(x));
          const int b = bin_of(x);
          atomicAdd(&s.hc[b], 1u);
          atomicAdd(&s.hl[b], (uint32_t)full & 0xffffu);
          atomicAdd(&s.hh[b], (uint32_t)(full >> 16));
        }
      }
    }
    cluster.sync();
    for (int i = rank * (NB / C) + tid; i < (rank + 1) * (NB / C); i += NT) {
      uint32_t c = 0;
      u64 m = 0;
      for (int o = 0; o < C; ++o) {
        c += cluster.map_shared_rank(s.hc, o)[i];
        m += cluster.map_shared_rank(s.hl, o)[i] + ((u64)cluster.map_shared_rank(s.hh, o)[i] << 16);
      }
      for (int o = 0; o < C; ++o) {
        cluster.map_shared_rank(s.gc, o)[i] = c;
        cluster.map_shared_rank(s.gm, o)[i] = m;
      }
    }
    cluster.sync();

    // 4  the element at which the running count (or weight), from the largest
    // element down, reaches `target`: its rank word; *mass: weight up to it
    auto find = [&](bool count, u64 target, int buf, u64 *mass) -> u64 {
      u64 before, other;
      const int b = count ? crossing<NB>(s, target, [&](int i) { return (u64)s.gc[i]; }, &before)
                          : crossing<NB>(s, target, [&](int i) { return s.gm[i]; }, &before);
      if (b >= NB) {  // fewer elements have a weight: all are kept
        *mass = reduce((u64)(s.gm[2 * tid] + s.gm[2 * tid + 1]), add, s.red);
        return 0;
      }
      {  // the other measure before the bin
        u64 o = 0;
        for (int i = tid; i < b; i += NT) o += count ? s.gm[i] : (u64)s.gc[i];
        other = reduce(o, add, s.red);
      }
      u64 acc_w = count ? other : before, acc = before;  // weight, and the target's measure, before the range
      const uint32_t k_lo = bin_end(b), k_hi = b ? bin_end(b - 1) - 1 : kmax;
      u64 lo = rank_word(k_lo, (int)MAX_VOCAB - 1), hi = rank_word(k_hi, 0);  // range of rank words
      const float x_lo = fmaxf(of_key(k_lo), cut), x_hi = of_key(k_hi);
      uint32_t cnt = s.gc[b];
      uint32_t mine_before = 0;  // elements of the range in lower ranks
      if (cnt <= CAP) {
        for (int o = 0; o < rank; ++o) mine_before += cluster.map_shared_rank(s.hc, o)[b];
      }
      while (cnt > CAP) {
        // narrow the range over the whole cluster, NB parts at a time
        const int shift = max(0, 64 - __clzll(hi - lo) - 10);
        cluster.sync();  // earlier reads of the narrowing bins are done
        for (int i = tid; i < NB; i += NT) s.nc[i] = s.nl[i] = s.nh[i] = 0;
        __syncthreads();
        for (int v = v0 + lane; v < v1; v += 32) {
          const uint4 q = xv[v];
          for (int j = 0; j < VEC; ++j) {
            const float x = get(q, j);
            if (x < x_lo || !(x <= x_hi)) continue;
            const u64 word = rank_word(key_of(x), i0 + v * VEC + j);
            if (word < lo || word > hi) continue;
            const int i = (int)((hi - word) >> shift);
            const u64 w = Row::w(f.e(x));
            atomicAdd(&s.nc[i], 1u);
            atomicAdd(&s.nl[i], (uint32_t)w & 0xffffu);
            atomicAdd(&s.nh[i], (uint32_t)(w >> 16));
          }
        }
        cluster.sync();
        auto all_c = [&](int i) {
          u64 c = 0;
          for (int o = 0; o < C; ++o) c += cluster.map_shared_rank(s.nc, o)[i];
          return c;
        };
        auto all_w = [&](int i) {
          u64 w = 0;
          for (int o = 0; o < C; ++o)
            w += cluster.map_shared_rank(s.nl, o)[i] + ((u64)cluster.map_shared_rank(s.nh, o)[i] << 16);
          return w;
        };
        u64 in;
        const int part = count ? crossing<NB>(s, target - acc, all_c, &in) : crossing<NB>(s, target - acc, all_w, &in);
        u64 o = 0;
        for (int i = tid; i < part; i += NT) o += all_w(i);
        acc_w += reduce(o, add, s.red);
        acc += in;
        hi -= (u64)part << shift;
        const u64 width = ((u64)1 << shift) - 1;
        lo = hi - lo > width ? hi - width : lo;
        cnt = (uint32_t)all_c(part);
        mine_before = 0;
        for (int o = 0; o < rank; ++o) mine_before += cluster.map_shared_rank(s.nc, o)[part];
      }
      // the range's elements, to every CTA of the cluster
      if (tid == 0) s.n_list = 0;
      __syncthreads();
      for (int v = v0 + lane; v < v1; v += 32) {
        const uint4 q = xv[v];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float x = get(q, j);
          if (!(x >= x_lo) || x > x_hi) continue;
          const u64 word = rank_word(key_of(x), i0 + v * VEC + j);
          if (word < lo || word > hi) continue;
          const int at = (int)mine_before + atomicAdd(&s.n_list, 1);
          const u64 w = Row::w(f.e(x));
          for (int o = 0; o < C; ++o) {
            cluster.map_shared_rank(s.list[buf], o)[at] = word;
            cluster.map_shared_rank(s.lw[buf], o)[at] = w;
          }
        }
      }
      cluster.sync();
      const u64 *list = s.list[buf], *lw = s.lw[buf];
      const int total = (int)cnt;
      while (cnt > FEW) {  // narrow the range within the list
        u64 mn = ~0ull, mx = 0;
        for (int i = tid; i < total; i += NT)
          if (list[i] >= lo && list[i] <= hi) {
            mn = min(mn, list[i]);
            mx = max(mx, list[i]);
          }
        lo = reduce(mn, low, s.red);
        hi = reduce(mx, high, s.red2);
        const int shift = max(0, 64 - __clzll(hi - lo) - 10);
        for (int i = tid; i < NB; i += NT) s.nc[i] = s.nl[i] = s.nh[i] = 0;
        __syncthreads();
        for (int i = tid; i < total; i += NT)
          if (list[i] >= lo && list[i] <= hi) {
            const int at = (int)((hi - list[i]) >> shift);
            atomicAdd(&s.nc[at], 1u);
            atomicAdd(&s.nl[at], (uint32_t)lw[i] & 0xffffu);
            atomicAdd(&s.nh[at], (uint32_t)(lw[i] >> 16));
          }
        __syncthreads();
        auto part_w = [&](int i) { return s.nl[i] + ((u64)s.nh[i] << 16); };
        u64 in;
        const int part = count ? crossing<NB>(s, target - acc, [&](int i) { return (u64)s.nc[i]; }, &in)
                               : crossing<NB>(s, target - acc, part_w, &in);
        u64 o = 0;
        for (int i = tid; i < part; i += NT) o += part_w(i);
        acc_w += reduce(o, add, s.red);
        acc += in;
        hi -= (u64)part << shift;
        const u64 width = ((u64)1 << shift) - 1;
        lo = hi - lo > width ? hi - width : lo;
        cnt = s.nc[part];
        __syncthreads();
      }
      if (tid == 0) s.n_list = 0;
      __syncthreads();
      for (int i = tid; i < total; i += NT)
        if (list[i] >= lo && list[i] <= hi) {
          const int at = atomicAdd(&s.n_list, 1);
          s.few[at] = list[i];
          s.few_w[at] = lw[i];
        }
      __syncthreads();
      const int few = s.n_list;
      if (tid < few) {
        const u64 me = s.few[tid], w = s.few_w[tid];
        u64 c = 0, m = 0;
        for (int j = 0; j < few; ++j)
          if (s.few[j] > me) {
            ++c;
            m += s.few_w[j];
          }
        const u64 ex = acc + (count ? c : m), own = count ? 1 : w;
        if (ex < target && target <= ex + own) {
          s.out_b = me;
          s.out_c = acc_w + m + w;
        }
      }
      __syncthreads();
      *mass = s.out_c;
      return s.out_b;
    };

    u64 W;
    if (by_count) thr = find(true, (u64)k, 0, &W);
    else W = reduce((u64)(s.gm[2 * tid] + s.gm[2 * tid + 1]), add, s.red);
    if (by_mass) {
      const double want = (double)p * (double)W;
      u64 dummy;
      const u64 t = find(false, want >= 1.0 ? (u64)want : 1, 1, &dummy);
      thr = max(thr, t);
    }
  }

  // 5  kept weight, in index order
  const uint32_t thr_key = (uint32_t)(thr >> IDX_BITS);
  const int thr_idx = (int)(MAX_VOCAB - 1 - (thr & (MAX_VOCAB - 1)));  // of the elements equal to it, up to this index
  if (thr) cut = fmaxf(cut, of_key(thr_key));
  if (pmin > 0.f) cut = fmaxf(cut, of_key(key_pmin));
  const float tie = thr ? of_key(thr_key) : -INFINITY;
  auto kept = [&](float x, int i) -> u64 {  // weight of element i, 0 if it is not kept
    if (!(x >= cut) || (x == tie && i > thr_idx)) return 0;
    return Row::w(f.e(x));
  };
  u64 sum = 0;
  for (int v = v0 + lane; v < v1; v += 32) {
    const uint4 q = xv[v];
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum += kept(get(q, j), i0 + v * VEC + j);
  }
#pragma unroll
  for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
  __syncthreads();
  if (lane == 0) s.red[warp] = sum;
  __syncthreads();
  u64 mine = 0, before = 0;
  for (int w = 0; w < NW; ++w) {
    if (w == warp) before = mine;
    mine += s.red[w];
  }
  if (tid < C) cluster.map_shared_rank(s.sums, tid)[rank] = mine;
  cluster.sync();
  u64 total = 0;
  for (int c = 0; c < C; ++c) {
    if (c == rank) before += total;
    total += s.sums[c];
  }
  const float u = a.u[r];
  u64 at = (u64)((double)(u > 0.f ? u : 0.f) * (double)total);
  at = at < total ? at : total - 1;
  if (before <= at && at < before + sum) {
    for (int v = v0; v < v1; v += 32) {
      const uint4 q = v + lane < v1 ? xv[v + lane] : make_uint4(0, 0, 0, 0);
      u64 own = 0;
      if (v + lane < v1) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) own += kept(get(q, j), i0 + (v + lane) * VEC + j);
      }
      u64 x = own;
#pragma unroll
      for (int w = 1; w < 32; w <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, x, w);
        if (lane >= w) x += y;
      }
      const uint32_t over = __ballot_sync(0xffffffffu, before + x > at);
      if (over) {
        if (lane == __ffs(over) - 1) {
          u64 c = before + x - own;
          int j = 0;
          for (; j < VEC - 1; ++j) {
            c += kept(get(q, j), i0 + (v + lane) * VEC + j);
            if (c > at) break;
          }
          a.tokens[r] = i0 + (v + lane) * VEC + j;
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, x, 31);
    }
  }
}

template <class T>
int launch_cluster(const Args &a, int slice, cudaStream_t st, int device) {
  const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + (size_t)slice * sizeof(T);
  static ContextOnce attr;
  if (int s = attr.run(device, []() -> int {
        NKB_CUDA_TRY(cudaFuncSetAttribute(cluster_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
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
  NKB_CUDA_TRY(cudaLaunchKernelEx(&cfg, cluster_kernel<T>, a, slice));
  return launch_status("sample_tokens");
}

// elements per CTA; 0 where a row does not fit a cluster
int slice_of(const Args &a) {
  const int64_t n = ((a.vocab + C - 1) / C + 7) / 8 * 8;
  const bool fits = n <= MAX_SLICE && (sizeof(Shared) + 15) / 16 * 16 + n * dtype_size((int)a.dtype) <= 227 * 1024;
  return fits ? (int)n : 0;
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
  const Row f{of_key(kmax), 1.f / temp};

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
    const double want = (double)p * (double)W;
    const u64 T = want >= 1.0 ? (u64)want : 1;
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
  const double x = (double)(a.u[r] > 0.f ? a.u[r] : 0.f) * (double)total;
  u64 at = (u64)x;
  at = at < total ? at : total - 1;
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
  if (a.rows < 0 || a.rows > INT32_MAX / C || a.vocab < 1) return bad("rows or vocab out of range");
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
  if (const int slice = slice_of(a)) {
    if (a.dtype == NKB_F32) return launch_cluster<float>(a, slice, st, device);
    if (a.dtype == NKB_BF16) return launch_cluster<__nv_bfloat16>(a, slice, st, device);
    return launch_cluster<__half>(a, slice, st, device);
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
