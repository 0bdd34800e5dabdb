// Appends new tokens' keys and values to a paged cache, rotating keys and
// queries on the way:
//   lo' = lo cos_p - hi sin_p,  hi' = lo sin_p + hi cos_p
// for the two halves (lo, hi) of the first rot_dim dimensions at position p,
// in fp32, rounded once to the stored type.  Each row is read and written once, so
// the bound is HBM.  Measured (GPU time): 8192 tokens of 32 + 2 * 8 rows of 128 bf16,
// 202 MB, 40.4 us or 5.0 TB/s, where a plain copy would take 31 us; 1500 tokens of
// 12 + 2 * 4 rows of 64 fp16 4.4 us, 8 tokens 2.2 us, which is the launch.
#include <algorithm>

#include "paged.cuh"

namespace nkb {
namespace append {

using Args = nkb_paged_append_args;

constexpr int THREADS = 256;

// Where a token goes: its sequence, the row of the rotation tables, and the
// offsets of its cache rows (-1: not stored).
struct Place {
  int seq;
  int64_t rope, k, v;
};
__device__ __forceinline__ Place place_of(const Args &a, int t, int b) {
  Place p = {b, 0, -1, -1};
  if (b < 0) return p;
  const int first = a.q_start ? a.q_start[b] : t, n = a.q_start ? a.q_start[b + 1] - first : 1;
  const int64_t pos = (int64_t)a.kv_len[b] - n + (t - first);
  if (pos >= 0 && pos < a.table_width * a.page_size) {
    const int i = (int)pos / (int)a.page_size, slot = (int)pos - i * (int)a.page_size;
    const int page = a.page_table[b * a.table_stride + i];
    if (paged::page_ok(page, a.pages)) {
      p.k = page * a.k_page + slot * a.k_slot;
      p.v = page * a.v_page + slot * a.v_slot;
    }
  }
  p.rope = max((int64_t)0, min(pos + a.pos_offset, a.rope_rows - 1)) * a.rope_stride;
  return p;
}

// Any layout: one block per token, its rows (query heads, key heads, value
// heads) element by element.
template <class T, class C>
__global__ void __launch_bounds__(THREADS) append_any_kernel(const __grid_constant__ Args a) {
  __shared__ int found;
  const int t = blockIdx.x;
  const Place at = place_of(a, t, paged::block_find_seq(a.q_start, (int)a.seqs, t, &found));
  const T *q = static_cast<const T *>(a.q), *k = static_cast<const T *>(a.k), *v = static_cast<const T *>(a.v);
  T *qo = static_cast<T *>(a.q_out);
  C *kc = static_cast<C *>(a.k_cache), *vc = static_cast<C *>(a.v_cache);
  const int D = (int)a.head_dim, half = (int)a.rot_dim / 2;
  const int hq = a.q_out ? (int)a.q_heads : 0, hkv = (int)a.kv_heads;
  for (int i = threadIdx.x; i < (hq + 2 * hkv) * D; i += THREADS) {
    const int h = i / D, d = i % D;
    if (h >= hq + hkv) {
      const int hv = h - hq - hkv;
      if (at.v >= 0)
        vc[at.v + hv * a.v_cache_head + d] = paged::from_f32<C>(paged::to_f32(v[t * a.v_token + hv * a.v_head + d]));
      continue;
    }
    const bool is_q = h < hq;
    const T *src = is_q ? q + t * a.q_token + h * a.q_head : k + t * a.k_token + (h - hq) * a.k_head;
    if (d >= half && d < 2 * half) continue;  // written with its partner
    float x = paged::to_f32(src[d]), y = 0.f;
    if (d < half) {
      const float hi = paged::to_f32(src[d + half]), c = load_as_float(a.cos, at.rope + d, (int)a.rope_dtype),
                  s = load_as_float(a.sin, at.rope + d, (int)a.rope_dtype);
      y = x * s + hi * c;
      x = x * c - hi * s;
    }
    if (is_q) {
      T *dst = qo + t * a.q_out_token + h * a.q_out_head;
      dst[d] = paged::from_f32<T>(at.seq < 0 ? 0.f : x);
      if (d < half) dst[d + half] = paged::from_f32<T>(at.seq < 0 ? 0.f : y);
    } else if (at.k >= 0) {
      C *dst = kc + at.k + (h - hq) * a.k_cache_head;
      dst[d] = paged::from_f32<C>(x);
      if (d < half) dst[d + half] = paged::from_f32<C>(y);
    }
  }
}

// Eight elements of a 16-byte piece (two pieces for fp32).
template <class T>
struct Eight {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4 *>(p)[i];
  }
  __device__ __forceinline__ void store(T *p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(p)[i] = w[i];
  }
  __device__ __forceinline__ void get(float *f) const {
    const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = paged::to_f32(e[i]);
  }
  __device__ __forceinline__ void set(const float *f) {
    T *e = reinterpret_cast<T *>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = paged::from_f32<T>(f[i]);
  }
};

// Rows of whole 16-byte pieces whose halves are whole pieces too: a row is
// `pieces` pairs of eight elements (d, d + rot_dim / 2 of the rotated part, then
// neighbouring pieces of the rest), one pair per thread and step.  Each byte is
// moved once; a block takes one token, so its place is looked up once, while
// the first rows are already on their way.  What a block waits for is the chain from
// its sequence over the length to the page, hidden by the other blocks of the SM:
// the more fit, the better.  With 256 threads for every token, some of them without
// a row, the 8192 tokens took 47.5 us and the 1500 6.9; so, two rows on the way per
// thread took as long, two to eight tokens per block 51 to 56 us, streaming loads and
// stores 46 to 50, and the stored rows would be gone from L2 when attention reads them.
template <class T, class C, class R>
__global__ void __launch_bounds__(THREADS) append_kernel(const __grid_constant__ Args a, int pieces, int unit) {
  __shared__ int found;
  const int t = blockIdx.x, half = (int)a.rot_dim / 2, D = (int)a.head_dim;
  const int hq = a.q_out ? (int)a.q_heads : 0, hkv = (int)a.kv_heads, rows = hq + 2 * hkv;
  const int step = blockDim.x / unit, c = threadIdx.x % unit, h0 = threadIdx.x / unit + blockIdx.y * step;
  const bool live = c < pieces && h0 < rows;
  const bool turns = c * 8 < half;
  // the pair's elements: d0 .. d0 + 7 and d1 .. d1 + 7 (none past the row's end)
  const int d0 = turns ? c * 8 : 2 * half + (c - half / 8) * 16, d1 = turns ? d0 + half : d0 + 8;
  const bool two = d1 < D;
  auto source = [&](int h) {
    return h < hq ? static_cast<const T *>(a.q) + t * a.q_token + h * a.q_head
           : h < hq + hkv ? static_cast<const T *>(a.k) + t * a.k_token + (h - hq) * a.k_head
                          : static_cast<const T *>(a.v) + t * a.v_token + (h - hq - hkv) * a.v_head;
  };
  Eight<T> lo, hi;
  if (live) {
    const T *src = source(h0);
    lo.load(src + d0);
    if (two) hi.load(src + d1);
  }
  const Place at = place_of(a, t, paged::block_find_seq(a.q_start, (int)a.seqs, t, &found));
  float cs[8], sn[8];
  if (live && turns) {
    Eight<R> e;
    e.load(static_cast<const R *>(a.cos) + at.rope + d0);
    e.get(cs);
    e.load(static_cast<const R *>(a.sin) + at.rope + d0);
    e.get(sn);
  }
  for (int h = h0; live && h < rows;) {
    float x[8], y[8];
    lo.get(x);
    hi.get(y);
    const int now = h;
    h += step * gridDim.y;
    if (h < rows) {  // the next row is on its way
      const T *src = source(h);
      lo.load(src + d0);
      if (two) hi.load(src + d1);
    }
    if (turns && now < hq + hkv) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = x[i], q = y[i];
        x[i] = p * cs[i] - q * sn[i];
        y[i] = p * sn[i] + q * cs[i];
      }
    }
    if (now < hq) {
      if (at.seq < 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.f;
      }
      Eight<T> o;
      T *dst = static_cast<T *>(a.q_out) + t * a.q_out_token + now * a.q_out_head;
      o.set(x);
      o.store(dst + d0);
      o.set(y);
      if (two) o.store(dst + d1);
    } else {
      const bool is_k = now < hq + hkv;
      const int64_t row = is_k ? at.k : at.v;
      if (row < 0) continue;
      C *dst = is_k ? static_cast<C *>(a.k_cache) + row + (now - hq) * a.k_cache_head
                    : static_cast<C *>(a.v_cache) + row + (now - hq - hkv) * a.v_cache_head;
      Eight<C> o;
      o.set(x);
      o.store(dst + d0);
      o.set(y);
      if (two) o.store(dst + d1);
    }
  }
}

// Whether every row starts at a 16-byte boundary and is made of whole pieces,
// the rotated halves too.
bool pieces_form(const Args &a) {
  const int64_t ts = dtype_size((int)a.dtype), cs = dtype_size((int)a.cache_dtype), rs = dtype_size((int)a.rope_dtype);
  auto whole = [](int64_t stride, int64_t size) { return stride >= 0 && stride * size % 16 == 0; };
  for (int64_t s : {a.k_token, a.k_head, a.v_token, a.v_head, a.q_token, a.q_head, a.q_out_token, a.q_out_head})
    if (!whole(s, ts)) return false;
  for (int64_t s : {a.k_page, a.k_slot, a.k_cache_head, a.v_page, a.v_slot, a.v_cache_head})
    if (!whole(s, cs)) return false;
  if (a.rot_dim && !whole(a.rope_stride, rs)) return false;
  uintptr_t p = 0;
  for (const void *x : {a.k, a.v, a.q, (const void *)a.q_out, (const void *)a.k_cache, (const void *)a.v_cache, a.cos, a.sin})
    p |= reinterpret_cast<uintptr_t>(x);
  return p % 16 == 0 && a.head_dim % 8 == 0 && a.rot_dim % 16 == 0 && a.head_dim <= 16 * THREADS;
}

int check_args(const Args &a) {
  auto bad = [](const char *m) { return fail(NKB_ERR_INVALID, std::string("paged_append: ") + m); };
  if (int s = paged::check_cache("paged_append", a.tokens, a.seqs, a.kv_heads, a.head_dim, a.pages, a.page_size,
                                 a.table_width, a.table_stride))
    return s;
  if (!paged::float_dtype(a.dtype) || !paged::float_dtype(a.cache_dtype))
    return fail(NKB_ERR_UNSUPPORTED, "paged_append: rows and caches must be float32, bfloat16 or float16");
  if (a.rot_dim < 0 || a.rot_dim % 2 || a.rot_dim > a.head_dim) return bad("rot_dim must be even and at most head_dim");
  if (a.rot_dim && (!a.cos || !a.sin || a.rope_rows < 1 || !paged::float_dtype(a.rope_dtype)))
    return bad("rotating needs cos and sin tables of a float type");
  // (an array without elements may be NULL, so a call without tokens says nothing by its pointers)
  if (a.q_heads < 0 || a.q_heads > 65535 ||
      (a.tokens && ((a.q_heads > 0) != (a.q_out != nullptr) || (a.q != nullptr) != (a.q_out != nullptr))))
    return bad("q, q_out and q_heads go together");
  if (a.tokens && (!a.k || !a.v || !a.kv_len || (a.table_width && !a.page_table) || (a.pages && (!a.k_cache || !a.v_cache))))
    return bad("NULL array");
  if (!a.q_start && a.tokens != a.seqs) return bad("without q_start there is one token per sequence");
  return NKB_OK;
}

int run(const Args &a, cudaStream_t st, int device) {
  if (int s = check_args(a)) return s;
  if (a.tokens == 0) return NKB_OK;
  if (!pieces_form(a)) {
    paged::with_dtype(a.dtype, [&](auto t) {
      return paged::with_dtype(a.cache_dtype, [&](auto c) {
        append_any_kernel<decltype(t), decltype(c)><<<(unsigned)a.tokens, THREADS, 0, st>>>(a);
        return 0;
      });
    });
    return launch_status("paged_append");
  }
  // pairs of pieces per row, and the threads that a row takes: the next power of two
  const int pieces = (int)(a.rot_dim / 16 + (a.head_dim - a.rot_dim + 15) / 16);
  int unit = 1;
  while (unit < pieces) unit *= 2;
  // a few tokens spread their rows over more blocks, of a warp at least; no more
  // threads than a block's rows need, in as many steps as a full block would take
  const int64_t rows = (a.q_out ? a.q_heads : 0) + 2 * a.kv_heads;
  const int64_t want = (2 * num_sms(device) + a.tokens - 1) / a.tokens;
  const int64_t split = std::max<int64_t>(1, std::min<int64_t>((rows * unit + 31) / 32, want));
  const int64_t per = (rows + split - 1) / split, steps = (per * unit + THREADS - 1) / THREADS;
  const unsigned threads = (unsigned)(((per + steps - 1) / steps * unit + 31) / 32 * 32);
  paged::with_dtype(a.dtype, [&](auto t) {
    return paged::with_dtype(a.cache_dtype, [&](auto c) {
      return paged::with_dtype(a.rot_dim ? a.rope_dtype : NKB_F32, [&](auto r) {
        append_kernel<decltype(t), decltype(c), decltype(r)><<<dim3((unsigned)a.tokens, (unsigned)split), threads, 0, st>>>(a, pieces, unit);
        return 0;
      });
    });
  });
  return launch_status("paged_append");
}

// "paged_append": the pointers of nkb_paged_append_args that are given; ints a
// mask of them and the struct's integers
int check(const Step &s) {
  Args a;
  if (int e = paged::step_args(s, nullptr, 11, 30, "paged_append", &a)) return e;
  return check_args(a);
}
int launch(const LaunchArgs &l) {
  Args a;
  if (int e = paged::step_args(*l.step, l.ptrs, 11, 30, "paged_append", &a)) return e;
  return run(a, l.stream, l.device);
}

}  // namespace append

NKB_REGISTER_KERNEL("paged_append", append::launch, append::check);

}  // namespace nkb

extern "C" int nkb_paged_append(const nkb_paged_append_args *args, void *stream) {
  if (!args) return nkb::fail(NKB_ERR_INVALID, "args is NULL");
  int dev = 0;
  cudaGetDevice(&dev);
  return nkb::append::run(*args, static_cast<cudaStream_t>(stream), dev);
}
