// Draws one token per row of logits: temperature, top-k, top-p and min-p, then
// the inverse of the kept weights' running sum at u.
//
// Weights are w = floor(2^32 exp((x - max) / temperature)): whole numbers, so
// every sum below is exact and independent of its order, whatever the number
// of threads.  A logit's key is the order-preserving image of its fp32 value
// (-0 as +0, NaN as -inf).  The kept set is described by a threshold key, the
// number of elements equal to it that are kept (in index order) and min_p.
#include "common.cuh"

namespace nkb {
namespace sample {

using Args = nkb_sample_args;
using u64 = unsigned long long;

constexpr int THREADS = 1024;

__device__ __forceinline__ float load_x(const void *p, int64_t i, int dt) {
  float x = __uint_as_float(load_as_reg(p, i, dt));
  if (x != x) x = -INFINITY;
  return x + 0.f;  // -0 becomes +0
}
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t KEY_NEG_INF = 0x007fffffu;  // key_of(-inf)

struct Row {
  float max, inv;  // largest logit, 1 / temperature
  __device__ __forceinline__ float e(float x) const {
    return x == max ? 1.f : x == -INFINITY ? 0.f : expf(__fmul_rn(__fsub_rn(x, max), inv));
  }
  static __device__ __forceinline__ u64 w(float e) { return (u64)(e * 4294967296.f); }
};

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

__global__ void __launch_bounds__(THREADS) sample_kernel(const __grid_constant__ Args a) {
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
  const Row f{__uint_as_float(kmax & 0x80000000u ? kmax & 0x7fffffffu : ~kmax), 1.f / temp};

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
    const u64 wt = Row::w(f.e(__uint_as_float(t & 0x80000000u ? t & 0x7fffffffu : ~t)));
    const u64 q = wt ? (T - above + wt - 1) / wt : ~0ull;
    quota = t == tau ? (q < quota ? q : quota) : q;
    tau = t;
  }
  float pmin = a.min_p ? a.min_p[r] : 0.f;
  pmin = pmin > 1.f ? 1.f : pmin;

  // kept weight of each warp's contiguous part: sum above tau and ties
  const int part = ((V + 31) / 32 + 31) / 32 * 32, i0 = warp * part, i1 = min(i0 + part, V);
  const float xt = __uint_as_float(tau & 0x80000000u ? tau & 0x7fffffffu : ~tau);
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

int run(const Args &a, cudaStream_t st) {
  auto bad = [](const char *m) { return fail(NKB_ERR_INVALID, std::string("sample_tokens: ") + m); };
  if (a.rows < 0 || a.rows > INT32_MAX || a.vocab < 1) return bad("rows or vocab out of range");
  if (a.dtype != NKB_F32 && a.dtype != NKB_BF16 && a.dtype != NKB_F16)
    return fail(NKB_ERR_UNSUPPORTED, "sample_tokens: logits must be float32, bfloat16 or float16");
  if (a.vocab > (1 << 21)) return fail(NKB_ERR_UNSUPPORTED, "sample_tokens: more than 2^21 entries");
  if (a.rows && (!a.logits || !a.u || !a.tokens)) return bad("NULL array");
  if (a.rows > 1 && a.row_stride < a.vocab) return bad("rows overlap");
  if (a.rows == 0) return NKB_OK;
  sample_kernel<<<(unsigned)a.rows, THREADS, 0, st>>>(a);
  return launch_status("sample_tokens");
}

}  // namespace sample
}  // namespace nkb

extern "C" int nkb_sample_tokens(const nkb_sample_args *args, void *stream) {
  if (!args) return nkb::fail(NKB_ERR_INVALID, "args is NULL");
  return nkb::sample::run(*args, static_cast<cudaStream_t>(stream));
}
