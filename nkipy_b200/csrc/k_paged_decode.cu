// Paged attention of one new token per sequence (bf16, fp16):
//   out[b, h] = sum_j softmax_j(q[b, h] . k_j * scale) v_j
// over the keys that the token sees, read once from their pages.
//
// The bound is HBM (4 G flop per 2-byte element of K and V for G query heads
// per key head), so the keys of all sequences are cut into equal shares: the
// sequences' key blocks, in (sequence, key head) order, form one run that the
// resident CTAs split evenly whatever the lengths.  A CTA therefore holds the
// end of one (sequence, key head), some whole ones, and the beginning of
// another; what it holds whole it writes out, the rest goes to a workspace as
// (max, sum, unnormalised output) for a second kernel to join.  Lengths are
// read on the device: the grid depends on none of them.
//
// A CTA's ring of stages goes on from one (sequence, key head) to the next, whose
// keys and query are loaded while the outputs of the one before are joined: with a
// ring that began anew at each, 8 sequences of 2048 keys took 22.3 us, 64 of 4100
// 175 us.  Two CTAs to an SM keep 128 KB on their way there.  Measured (32 / 8 heads
// of 128 bf16, GPU time with the join): 64 sequences of 4100 keys 172 us, 6.2 of the
// 6.5 TB/s of a copy; 8 of 2048 19.5 us, 3.5 TB/s: a share is seven blocks there, and
// before the first of them length, page and key are read one after another, after
// the last comes the join; one of 500 6.0 us.  The matrix units are far from busy.
//
// In a CTA the (up to 16) query heads of the key head are the rows of one m16
// tile; each of four warps takes every fourth group of WN keys through its own
// ring of stages filled by cp.async, scores and products on mma.sync m16n8k16
// with fp32 accumulation, the running maximum and sum of the softmax in fp32.
#include "mma_sync.cuh"
#include "paged_attn.cuh"

namespace nkb {
namespace pattn {
namespace {

using mma::cp_async16;
using mma::cp_commit;
using mma::cp_wait;
using mma::ldsm_x4;
using mma::ldsm_x4_t;
using mma::smem_addr;

using namespace single;

template <class T>
__device__ __forceinline__ void mma_tile(float *c, const uint32_t *a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_tile<__nv_bfloat16>(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
  mma::mma16816(c, a, b0, b1);
}
template <>
__device__ __forceinline__ void mma_tile<__half>(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <class T, int DP>
__global__ void __launch_bounds__(THREADS, 2) decode_kernel(const __grid_constant__ Params p) {
  using S = Shape<DP>;
  constexpr int WN = S::WN, NT = WN / 8, CH = DP / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *sQ = smem;
  const Args &a = p.a;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, c = blockIdx.x;
  const int heads = (int)a.kv_heads * p.groups;  // units per sequence
  const int G = (int)(a.q_heads / a.kv_heads), D = (int)a.head_dim;
  uint8_t *ring = smem + S::STAGES * S::QBUF + warp * S::RING;
  float2 *s_ml = reinterpret_cast<float2 *>(smem + S::STAGES * S::QBUF + WARPS * S::RING);  // (max, sum) of the warps' rows

  const Found at = find<S::BK>(a, [&](int64_t blocks, int, int64_t first, int64_t n) {
    const Split split(blocks * heads, p.ctas);
    const int64_t f = split.first(min(c, split.ctas - 1));
    return first * heads <= f && f < (first + n) * heads;
  });
  pdl_trigger();
  const Split split(at.total * heads, p.ctas);
  if (c >= split.ctas) {
    pdl_wait();
    return;
  }
  const int64_t f0 = split.first(c);
  const int n_blocks = (int)(split.first(c + 1) - f0);

  // a place in the share: block k of nb of a (sequence, 16-row group of heads)
  struct At {
    int b, unit, k, nb;
    Visible vis;
  };
  auto sequence = [&](At &x, int b) {
    x.b = b;
    x.vis = visible_of(a, b);
    x.nb = max(1, (x.vis.n + S::BK - 1) / S::BK);
  };
  auto step = [&](At &x) {
    if (++x.k < x.nb) return;
    x.k = 0;
    if (++x.unit < heads) return;
    x.unit = 0;
    if (x.b + 1 < (int)a.seqs) sequence(x, x.b + 1);
  };
  At ahead;  // of the next block to locate
  sequence(ahead, at.seq);
  {
    const int in = (int)(f0 - at.before * heads);
    ahead.unit = in / ahead.nb;
    ahead.k = in - ahead.unit * ahead.nb;
  }
  At now = ahead;  // of the block at work

  // where this lane's key of a located block and its value begin (null: no such
  // key or page), and the block's unit
  const char *k_row, *v_row;
  int unit_b, unit, located = 0;
  bool starts;  // the block is the first of its segment: Q goes with it
  auto locate = [&]() {
    k_row = v_row = nullptr;
    starts = ahead.k == 0 || located == 0;
    unit_b = ahead.b;
    unit = ahead.unit;
    if (located++ >= n_blocks) return;
    const int v = ahead.k * S::BK + warp * WN + lane;
    if (lane < WN && v < ahead.vis.n) {
      const int key = ahead.vis.key(v), i = key / (int)a.page_size, slot = key - i * (int)a.page_size;
      const int page = a.page_table[ahead.b * a.table_stride + i];
      if (paged::page_ok(page, a.pages)) {
        const int hk = p.groups == 1 ? unit : unit / p.groups;
        k_row = reinterpret_cast<const char *>(static_cast<const T *>(a.k_cache) + page * a.k_page + slot * a.k_slot +
                                               hk * a.k_cache_head);
        v_row = reinterpret_cast<const char *>(static_cast<const T *>(a.v_cache) + page * a.v_page + slot * a.v_slot +
                                               hk * a.v_cache_head);
      }
    }
    step(ahead);
  };
  int q_next = 0, q_at = 0;  // Q buffers: the next to fill, the one in use
  // the located block into `stage`; rows without a page are zeros
  auto load = [&](int stage) {
    const uint32_t kd = smem_addr(ring + stage * 2 * S::TILE), vd = kd + S::TILE;
#pragma unroll
    for (int j = 0; j < WN * CH / 32; ++j) {
      const int idx = j * 32 + lane, r = idx / CH, ch = idx % CH;
      const uint64_t k = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(k_row), r);
      const uint64_t v = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(v_row), r);
      const bool ok = k && ch * 8 < D;
      cp_async16(kd + mma::swz(r, ch, DP * 2), ok ? reinterpret_cast<const char *>(k) + ch * 16 : a.k_cache, ok);
      cp_async16(vd + mma::swz(r, ch, DP * 2), ok ? reinterpret_cast<const char *>(v) + ch * 16 : a.v_cache, ok);
    }
    if (starts) {  // each warp copies a quarter of the rows of Q
      const int hk = unit / p.groups, g0 = (unit - hk * p.groups) * ROWS, rows = min(ROWS, G - g0);
      const T *q = static_cast<const T *>(a.q) + unit_b * a.q_token + (hk * G + g0) * a.q_head;
      const uint32_t qd = smem_addr(sQ + q_next * S::QBUF);
#pragma unroll
      for (int j = 0; j < (ROWS / WARPS * CH + 31) / 32; ++j) {
        const int idx = j * 32 + lane, r = warp * (ROWS / WARPS) + idx / CH, ch = idx % CH;
        const bool ok = r < rows && ch * 8 < D;
        cp_async16(qd + mma::swz(r, ch, DP * 2), q + (ok ? r * a.q_head + ch * 8 : 0), ok);
      }
      q_next = q_next + 1 == S::STAGES ? 0 : q_next + 1;
    }
  };
  locate();
#pragma unroll
  for (int s = 0; s < S::STAGES - 1; ++s) {
    if (s < n_blocks) load(s);
    locate();
    cp_commit();
  }

  uint32_t qf[DP / 16][4];
  float o[CH][4], m[2], l[2];  // rows lane / 4 and lane / 4 + 8, log2 units
  int stage = 0, k0 = 0;  // k0: the segment's first block in its unit
  bool first = true;      // the next block starts one
#pragma unroll 1
  for (int i = 0; i < n_blocks; ++i) {
    __syncwarp();  // every lane has read the stage that is filled next
    {
      int fill = stage + S::STAGES - 1;
      fill = fill >= S::STAGES ? fill - S::STAGES : fill;
      if (i + S::STAGES - 1 < n_blocks) load(fill);
      locate();
      cp_commit();
    }
    cp_wait<S::STAGES - 1>();
    __syncwarp();  // this block's rows, copied by every lane, are visible
    uint8_t *tile = ring + stage * 2 * S::TILE;
    const uint32_t kt = smem_addr(tile), vt = kt + S::TILE;
    stage = stage + 1 == S::STAGES ? 0 : stage + 1;
    if (first) {
      __syncthreads();  // every warp's rows of Q
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
        ldsm_x4(smem_addr(sQ + q_at * S::QBUF) + mma::swz(lane % 16, kk * 2 + lane / 16, DP * 2), qf[kk][0], qf[kk][1],
                qf[kk][2], qf[kk][3]);
      q_at = q_at + 1 == S::STAGES ? 0 : q_at + 1;
#pragma unroll
      for (int j = 0; j < CH; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
      k0 = now.k;
      first = false;
    }
    float s[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
      for (int j = 0; j < NT; j += 2) {
        uint32_t b0, b1, b2, b3;
        const int r = j * 8 + (lane % 8) + (lane / 16) * 8;
        ldsm_x4(kt + mma::swz(r, kk * 2 + (lane / 8) % 2, DP * 2), b0, b1, b2, b3);
        mma_tile<T>(s[j], qf[kk], b0, b1);
        mma_tile<T>(s[j + 1], qf[kk], b2, b3);
      }
    const int v0 = now.k * S::BK + warp * WN;
    float mx[2] = {m[0], m[1]};
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = v0 + j * 8 + (lane % 4) * 2 + (e & 1);
        s[j][e] = v < now.vis.n ? s[j][e] * p.scale_log2 : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], s[j][e]);
      }
    float alpha[2], sum[2] = {0.f, 0.f}, base[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      base[i] = base_of(mx[i]);
      alpha[i] = ex2(m[i] - base[i]);
      m[i] = mx[i];
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[j][e] = ex2(s[j][e] - base[e >> 1]);
        sum[e >> 1] += s[j][e];
      }
    l[0] = l[0] * alpha[0] + sum[0];
    l[1] = l[1] * alpha[1] + sum[1];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      o[j][0] *= alpha[0];
      o[j][1] *= alpha[0];
      o[j][2] *= alpha[1];
      o[j][3] *= alpha[1];
    }
#pragma unroll
    for (int kk = 0; kk < NT / 2; ++kk) {
      // probabilities rounded to the cache's type, as the matrix product takes its operands in one type (the sums keep
      // fp32 ones): bf16 outputs are 0.0020 to 0.0022 from 64-bit values in the root mean square, 0.0017 with fp32 ones
      const uint32_t pf[4] = {pack<T>(s[2 * kk][0], s[2 * kk][1]), pack<T>(s[2 * kk][2], s[2 * kk][3]),
                              pack<T>(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack<T>(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
      for (int j = 0; j < CH; j += 2) {
        uint32_t b0, b1, b2, b3;
        const int r = kk * 16 + (lane % 8) + ((lane / 8) % 2) * 8;
        ldsm_x4_t(vt + mma::swz(r, j + lane / 16, DP * 2), b0, b1, b2, b3);
        mma_tile<T>(o[j], pf, b0, b1);
        mma_tile<T>(o[j + 1], pf, b2, b3);
      }
    }
    if (now.k + 1 < now.nb && i + 1 < n_blocks) {
      ++now.k;
      continue;
    }

    // the segment's end: join the four warps, in the stage that each has just read
    // (the others are being filled)
    const int hk = now.unit / p.groups, g0 = (now.unit - hk * p.groups) * ROWS, rows = min(ROWS, G - g0);
    auto at_o = [](int r, int d) { return r * DP + (d ^ ((r & 3) * 8)); };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = lane / 4 + i * 8;
      if (r >= rows) continue;
      if (lane % 4 == 0) s_ml[warp * ROWS + r] = make_float2(m[i], l[i]);
#pragma unroll
      for (int j = 0; j < CH; ++j)
        *reinterpret_cast<float2 *>(reinterpret_cast<float *>(tile) + at_o(r, j * 8 + (lane % 4) * 2)) =
            make_float2(o[j][2 * i], o[j][2 * i + 1]);
    }
    __syncthreads();
    const bool all = k0 == 0 && now.k + 1 == now.nb, whole = all && !p.keep;
    const int64_t at_slot = all ? 2 * p.ctas + (int64_t)now.b * heads + now.unit : 2 * c + (i + 1 > now.k + 1 - k0);
    float *slot_ws = p.ws + at_slot * S::SLOT;
    for (int i = threadIdx.x; i < rows * (DP / 4); i += THREADS) {
      const int r = i / (DP / 4), d = i % (DP / 4) * 4;
      float2 ml[WARPS];
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        ml[w] = s_ml[w * ROWS + r];
        M = fmaxf(M, ml[w].x);
      }
      float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float g = ml[w].x == -INFINITY ? 0.f : ex2(ml[w].x - M);
        const uint8_t *part = tile + (w - warp) * S::RING;
        const float4 y = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(part) + at_o(r, d));
        L += ml[w].y * g;
        x[0] += y.x * g;
        x[1] += y.y * g;
        x[2] += y.z * g;
        x[3] += y.w * g;
      }
      if (whole) {
        const float inv = inverse(L);
        if (d < D)
          *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + now.b * a.out_token + (hk * G + g0 + r) * a.out_head + d) =
              make_uint2(pack<T>(x[0] * inv, x[1] * inv), pack<T>(x[2] * inv, x[3] * inv));
      } else {
        *reinterpret_cast<float4 *>(slot_ws + r * DP + d) = make_float4(x[0], x[1], x[2], x[3]);
        if (d == 0) *reinterpret_cast<float2 *>(slot_ws + ROWS * DP + 2 * r) = make_float2(M, L);
      }
    }
    __syncthreads();  // the stages may be filled again
    step(now);
    first = true;
  }
  pdl_wait();  // launched early, this grid must not end before the one it follows
}

// Joins the partials of one (sequence, 16-row group of heads).
template <class T, int DP>
__global__ void __launch_bounds__(THREADS) decode_join_kernel(const __grid_constant__ Params p) {
  using S = Shape<DP>;
  const Args &a = p.a;
  const int heads = (int)a.kv_heads * p.groups, b = blockIdx.x / heads, unit = blockIdx.x % heads;
  const int G = (int)(a.q_heads / a.kv_heads), D = (int)a.head_dim;
  const int hk = unit / p.groups, h0 = hk * G + (unit % p.groups) * ROWS, rows = min(ROWS, (hk + 1) * G - h0);
  const Found at = find<S::BK>(a, [&](int64_t, int s, int64_t, int64_t) { return s == b; });
  const int nb = blocks_of<S::BK>(a, b);
  const int64_t first = at.before * heads + (int64_t)unit * nb;
  const Parts parts = parts_of(Split(at.total * heads, p.ctas), first, nb, p.ctas, blockIdx.x);
  pdl_wait();  // in every block: the grid must not end before the one it follows
  if (parts.n == 1 && !p.keep) return;  // one CTA held it whole
  for (int i = threadIdx.x; i < rows * (DP / 4); i += THREADS) {
    const int r = i / (DP / 4), d = i % (DP / 4) * 4;
    if (d >= D) continue;
    Joined<8> x;
    x.add(parts.n, [&](int j) {
      const float *slot = p.ws + (int64_t)parts.slot(j) * S::SLOT;
      return Partial{slot + r * DP + d, slot + ROWS * DP + 2 * r};
    });
    x.store(static_cast<T *>(a.out) + b * a.out_token + (h0 + r) * a.out_head + d);
  }
}

int grid_ctas(int device) { return 2 * num_sms(device); }

template <class T, int DP>
int launch(const Params &p, cudaStream_t st, int device, bool pdl) {
  static ContextOnce attr;
  if (int s = attr.run(device, []() -> int {
        NKB_CUDA_TRY(cudaFuncSetAttribute(decode_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP>::SMEM));
        return NKB_OK;
      }))
    return s;
  NKB_CUDA_TRY(launch_pdl(pdl, decode_kernel<T, DP>, dim3(p.ctas), dim3(THREADS), Shape<DP>::SMEM, st, p));
  if (int s = launch_status("paged_decode")) return s;
  if (p.keep) return NKB_OK;
  const int64_t units = p.a.seqs * p.a.kv_heads * p.groups;
  NKB_CUDA_TRY(launch_pdl(true, decode_join_kernel<T, DP>, dim3((unsigned)units), dim3(THREADS), 0, st, p));
  return launch_status("paged_decode join");
}

}  // namespace

size_t decode_workspace(const Args &a, int device, bool keep) {
  const int64_t groups = (a.q_heads / a.kv_heads + ROWS - 1) / ROWS;
  return (size_t)(2 * grid_ctas(device) + (keep ? a.seqs * a.kv_heads * groups : 0)) *
         (a.head_dim <= 64 ? Shape<64>::SLOT : Shape<128>::SLOT) * sizeof(float);
}

int decode_params(const Args &a, int device, void *workspace, bool keep, Params *p) {
  p->a = a;
  p->groups = (int)((a.q_heads / a.kv_heads + ROWS - 1) / ROWS);
  p->scale_log2 = (float)(a.scale * LOG2E);
  p->ws = static_cast<float *>(workspace);
  p->ctas = grid_ctas(device);
  p->keep = keep;
  return NKB_OK;
}

int decode_launch(const Params &p, cudaStream_t st, int device, bool pdl) {
  if (p.a.dtype == NKB_BF16)
    return p.a.head_dim <= 64 ? launch<__nv_bfloat16, 64>(p, st, device, pdl) : launch<__nv_bfloat16, 128>(p, st, device, pdl);
  return p.a.head_dim <= 64 ? launch<__half, 64>(p, st, device, pdl) : launch<__half, 128>(p, st, device, pdl);
}

}  // namespace pattn
}  // namespace nkb
