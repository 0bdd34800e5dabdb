// Appends new tokens' keys and values to a paged cache, rotating keys and
// queries on the way:
//   lo' = lo cos_p - hi sin_p,  hi' = lo sin_p + hi cos_p
// for the two halves (lo, hi) of the first rot_dim dimensions at position p,
// in fp32, rounded once to the stored type.
#include "paged.cuh"

namespace nkb {
namespace append {

using Args = nkb_paged_append_args;

constexpr int THREADS = 256;

// One block per token: its rows (query heads, key heads, value heads), element
// by element.
template <class T, class C>
__global__ void __launch_bounds__(THREADS) append_kernel(const __grid_constant__ Args a) {
  __shared__ int slot;
  const int t = blockIdx.x;
  const int b = paged::block_find_seq(a.q_start, (int)a.seqs, t, &slot);
  const T *q = static_cast<const T *>(a.q), *k = static_cast<const T *>(a.k), *v = static_cast<const T *>(a.v);
  T *qo = static_cast<T *>(a.q_out);
  C *kc = static_cast<C *>(a.k_cache), *vc = static_cast<C *>(a.v_cache);
  const int D = (int)a.head_dim, half = (int)a.rot_dim / 2;
  int64_t pos = 0, cache_row_k = -1, cache_row_v = -1;
  if (b >= 0) {
    const int first = a.q_start ? a.q_start[b] : t, n = a.q_start ? a.q_start[b + 1] - first : 1;
    pos = (int64_t)a.kv_len[b] - n + (t - first);
    if (pos >= 0 && pos < a.table_width * a.page_size) {
      const int page = a.page_table[b * a.table_stride + pos / a.page_size];
      if (paged::page_ok(page, a.pages)) {
        const int64_t s = pos % a.page_size;
        cache_row_k = page * a.k_page + s * a.k_slot;
        cache_row_v = page * a.v_page + s * a.v_slot;
      }
    }
  }
  int64_t row = pos + a.pos_offset;
  row = row < 0 ? 0 : row >= a.rope_rows ? a.rope_rows - 1 : row;
  auto angle = [&](const void *table, int i) {
    return load_as_float(table, row * a.rope_stride + i, (int)a.rope_dtype);
  };
  const int hq = a.q_out ? (int)a.q_heads : 0, hkv = (int)a.kv_heads;
  for (int i = threadIdx.x; i < (hq + 2 * hkv) * D; i += THREADS) {
    const int h = i / D, d = i % D;
    if (h >= hq + hkv) {
      const int hv = h - hq - hkv;
      if (cache_row_v >= 0)
        vc[cache_row_v + hv * a.v_cache_head + d] = paged::from_f32<C>(paged::to_f32(v[t * a.v_token + hv * a.v_head + d]));
      continue;
    }
    const bool is_q = h < hq;
    const T *src = is_q ? q + t * a.q_token + h * a.q_head : k + t * a.k_token + (h - hq) * a.k_head;
    if (d >= half && d < 2 * half) continue;  // written with its partner
    float x = paged::to_f32(src[d]), y = 0.f;
    if (d < half) {
      const float hi = paged::to_f32(src[d + half]), c = angle(a.cos, d), s = angle(a.sin, d);
      y = x * s + hi * c;
      x = x * c - hi * s;
    }
    if (is_q) {
      T *dst = qo + t * a.q_out_token + h * a.q_out_head;
      dst[d] = paged::from_f32<T>(b < 0 ? 0.f : x);
      if (d < half) dst[d + half] = paged::from_f32<T>(b < 0 ? 0.f : y);
    } else if (cache_row_k >= 0) {
      C *dst = kc + cache_row_k + (h - hq) * a.k_cache_head;
      dst[d] = paged::from_f32<C>(x);
      if (d < half) dst[d + half] = paged::from_f32<C>(y);
    }
  }
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
  if (a.q_heads < 0 || a.q_heads > 65535 || (a.q_heads > 0) != (a.q_out != nullptr) || (a.q != nullptr) != (a.q_out != nullptr))
    return bad("q, q_out and q_heads go together");
  if (a.tokens && (!a.k || !a.v || !a.kv_len || (a.table_width && !a.page_table) || (a.pages && (!a.k_cache || !a.v_cache))))
    return bad("NULL array");
  if (!a.q_start && a.tokens != a.seqs) return bad("without q_start there is one token per sequence");
  return NKB_OK;
}

int run(const Args &a, cudaStream_t st) {
  if (int s = check_args(a)) return s;
  if (a.tokens == 0) return NKB_OK;
  paged::with_dtype(a.dtype, [&](auto t) {
    return paged::with_dtype(a.cache_dtype, [&](auto c) {
      append_kernel<decltype(t), decltype(c)><<<(unsigned)a.tokens, THREADS, 0, st>>>(a);
      return 0;
    });
  });
  return launch_status("paged_append");
}

}  // namespace append
}  // namespace nkb

extern "C" int nkb_paged_append(const nkb_paged_append_args *args, void *stream) {
  if (!args) return nkb::fail(NKB_ERR_INVALID, "args is NULL");
  return nkb::append::run(*args, static_cast<cudaStream_t>(stream));
}
