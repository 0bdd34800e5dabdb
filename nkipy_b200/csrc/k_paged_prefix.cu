// Paged attention of a batch whose sequences share their first prefix_len
// tokens:
//   out[t, h] = softmax over (prefix keys, own keys) times their values.
// The prefix is attended once for all: the batch's tokens and the query heads
// of a key head are the rows of the tensor-core tiles (k_paged_tile.cu), so its
// keys and values are read once per 2 P tokens instead of once per sequence.
// Each sequence's own keys take the form for single tokens or for several, and
// both leave partials (max, sum, unnormalised output) that the kernel here
// joins per token and head.  Measured (32 / 8 heads of 128 bf16, GPU time): 64
// sequences with some hundred keys each after a prefix of 8192, 44 us (the floor is
// 14 us of reads; prefix 29 on two thirds of the SMs, own keys 21 and join 12 us one by
// one with cold caches, each in part under the next: few blocks per CTA, so each is
// mostly its start and its partials); 4 sequences after a prefix of 1000, 15.7 us.
#include "paged_attn.cuh"

namespace nkb {
namespace pattn {
namespace {

constexpr int THREADS = single::THREADS;
// Rows per SM up to which a block takes one.  28 tokens of 5 heads 36 us, shared 19;
// 56 of 8 28 and 25; 63 of 28 24 and 31, 64 of 32 56 and 63: more blocks, each with
// its start, cost more than the shorter chain of reads gives.
constexpr int FEW = 4;

// A group of DP / 4 threads reads a row's partials, four outputs a thread.  With few
// tokens all groups of the block share one row's partials (`share`), and a block has
// one query head; else each group has a query head of its own.
template <class T, int DP>
__global__ void __launch_bounds__(THREADS)
    prefix_join_kernel(const __grid_constant__ several::Params p, const __grid_constant__ single::Params s, int share) {
  constexpr int LANES = DP / 4, GROUPS = THREADS / LANES;
  __shared__ float4 s_x[THREADS];
  __shared__ float2 s_ml[THREADS];
  using S = single::Shape<DP>;
  constexpr int SLOT = several::slot_floats(DP), ML = 2 * several::BM * DP;
  const Args &a = p.a;
  const int t = blockIdx.x, hk = blockIdx.y, G = p.G, D = (int)a.head_dim, per = 2 * p.P;
  single::Found at = {0, 0, 0};
  if (p.own) pdl_wait();  // the pairs are a list of the kernels before
  else at = single::find<S::BK>(a, [&](int64_t, int b, int64_t, int64_t) { return b == t; });
  const several::Walk walk(p, 0);
  // of pair u; -2 where the token is not one of its own (a list of starts that go back, which no caller means, is cut
  // off at the pairs that there is room for)
  auto unit_parts = [&](int u, int &tok, int &seq) {
    const several::Pair x = walk.list.pair(u);
    const int64_t n = several::blocks_of(p, x).n;
    tok = t - x.tok0;
    seq = tok >= 0 && tok < x.ntok ? x.seq : -2;
    return walk.parts(u, hk, n);
  };
  int ptok, otok = 0, seq = 0;
  const Parts pre = unit_parts(t / per, ptok, seq);
  Parts own;
  seq = 0;
  if (p.own) {  // the pair of this token among the sequences' own
    int lo = (int)((a.tokens + per - 1) / per), hi = walk.pairs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (p.pairs[mid].tok0 <= t) lo = mid;
      else hi = mid - 1;
    }
    own = unit_parts(lo, otok, seq);
  }
  const int heads = (int)a.kv_heads * s.groups;
  auto own_parts = [&](int g) {
    const int unit = hk * s.groups + g / single::ROWS, nb = single::blocks_of<S::BK>(a, t);
    return parts_of(Split(at.total * heads, s.ctas), at.before * heads + (int64_t)unit * nb, nb, s.ctas, (int64_t)t * heads + unit);
  };
  const int group = threadIdx.x / LANES, d = threadIdx.x % LANES * 4, sub = group % share;
  const int g0 = blockIdx.z * (GROUPS / share) + group / share, step = gridDim.z * (GROUPS / share);
  if (!p.own) {
    own = own_parts(min(g0, G - 1));
    pdl_wait();
  }
  for (int g = g0; g < G; g += step) {  // (with share > 1 the same in all threads)
    if (!p.own && g != g0) own = own_parts(g);
    auto tile_part = [&](const Parts &x, int j, int tok) {
      const float *slot = p.ws + (int64_t)x.slot(j) * SLOT;
      const int row = tok / p.P * several::BM + tok % p.P * G + g;
      return Partial{slot + row * DP + d, slot + ML + 2 * row};
    };
    Joined<8> x;
    if (seq != -2) {  // (a token of no sequence sees nothing)
      auto mine = [&](int n) { return (n - sub + share - 1) / share; };
      x.add(mine(pre.n), [&](int j) { return tile_part(pre, sub + j * share, ptok); });
      if (p.own) x.add(mine(own.n), [&](int j) { return tile_part(own, sub + j * share, otok); });
      else
        x.add(mine(own.n), [&](int j) {
          const float *slot = s.ws + (int64_t)own.slot(sub + j * share) * S::SLOT;
          const int row = g % single::ROWS;
          return Partial{slot + row * DP + d, slot + single::ROWS * DP + 2 * row};
        });
    }
    if (share > 1) {
      __syncthreads();  // the row before is read
      s_x[threadIdx.x] = make_float4(x.x[0], x.x[1], x.x[2], x.x[3]);
      s_ml[threadIdx.x] = make_float2(x.m, x.l);
      __syncthreads();
      if (sub) continue;
      Joined<8> all;
      all.add_from(share, [&](int j) { return s_ml[threadIdx.x + j * LANES]; }, [&](int j) { return s_x[threadIdx.x + j * LANES]; });
      x = all;
    }
    if (d < D) x.store(static_cast<T *>(a.out) + t * a.out_token + (hk * G + g) * a.out_head + d);
  }
}

size_t up(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

size_t prefix_workspace(const Args &a, int device) {
  const bool own = a.q_start != nullptr;
  return up(tile_workspace(a, device, own, true, true)) + (own ? 0 : decode_workspace(a, device, true));
}

int prefix_run(const Args &a, cudaStream_t st, int device) {
  const bool own = a.q_start != nullptr;
  several::Params p;
  single::Params s = {};
  tile_params(a, device, a.workspace, own, true, true, &p);
  // Where the sequences' own keys have a kernel of their own, it begins on the SMs
  // that a short prefix leaves it: two thirds for the prefix, and fewer partials.  A
  // long prefix is then what takes the time, and gets all SMs.  32 / 8 heads of 128
  // bf16, us with two thirds and with all, for 50, 400 and 2000 own keys: 64 after
  // 2000 (1 block per CTA) 28, 43, 108 and 29, 46, 112; 64 after 8192 (3.5) 35, 54,
  // 128 and 34, 56, 124; 128 after 8192 (7) 54, 88, 213 and 51, 88, 218; 256 after 8192
  // (14) 99, 155, 400 and 92, 145, 409; 128 after 32768 (28) 118, 146, 264 and 97, 128, 260.
  if (!own) {
    const int64_t per = 2 * p.P, units = (a.tokens + per - 1) / per * a.kv_heads;
    if (units * ((a.prefix_len + several::BN - 1) / several::BN) <= 8 * (int64_t)p.max_ctas) p.max_ctas = max(1, p.max_ctas * 2 / 3);
  }
  decode_params(a, device, static_cast<char *>(a.workspace) + up(tile_workspace(a, device, own, true, true)), true, &s);
  if (int e = tile_launch(p, st, device)) return e;
  if (!own)
    if (int e = decode_launch(s, st, device, true)) return e;
  const bool bf16 = a.dtype == NKB_BF16, small = a.head_dim <= 64;
  const int64_t G = a.q_heads / a.kv_heads;
  const bool shared = a.tokens * a.kv_heads * G <= FEW * num_sms(device);
  const dim3 grid((unsigned)a.tokens, (unsigned)a.kv_heads, shared ? (unsigned)G : 1);
  const int share = shared ? THREADS / (small ? 16 : 32) : 1;
  auto join = [&](auto kernel) { return launch_pdl(true, kernel, grid, dim3(THREADS), 0, st, p, s, share); };
  NKB_CUDA_TRY(bf16 ? (small ? join(prefix_join_kernel<__nv_bfloat16, 64>) : join(prefix_join_kernel<__nv_bfloat16, 128>))
                    : (small ? join(prefix_join_kernel<__half, 64>) : join(prefix_join_kernel<__half, 128>)));
  return launch_status("paged prefix join");
}

}  // namespace pattn
}  // namespace nkb
