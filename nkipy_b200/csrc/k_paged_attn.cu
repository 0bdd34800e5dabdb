// Attention of new tokens over a paged cache, with a sliding window and first
// tokens that stay visible, or over a prefix that the batch shares:
//   out[t, h] = sum_j softmax_j(q[t, h] . k_j * scale) v_j
// over the keys j that the token at position p sees (j <= p, and with a window
// w also j > p - w or j < sinks; all of the prefix).
#include <cfloat>
#include <cmath>

#include "paged_attn.cuh"

namespace nkb {
namespace pattn {

constexpr int WARPS = 4, MAX_D = 256;

// Any type, layout, page size and head dimension up to 256: one block per
// (token, query head), its four warps taking every fourth key; lane l holds
// dimensions l, l + 32, ... of the query, the running output and each row, so
// a score is a warp sum.  Running maximum and sum per warp (fp32), joined at
// the end.  Bound by the instructions per key (a warp sum each): 8 sequences of
// 2048 keys, 32 / 8 heads of 128 bf16, take 465 us, 20 in the form for rows of
// 16-byte pieces; it is for what the other forms cannot take.
template <class T>
__global__ void __launch_bounds__(WARPS * 32) attn_any_kernel(const __grid_constant__ Args a) {
  constexpr int PER = MAX_D / 32;
  __shared__ int slot;
  __shared__ float s_m[WARPS], s_l[WARPS], s_o[WARPS][MAX_D];
  const int t = blockIdx.x, h = blockIdx.y, hk = h / (int)(a.q_heads / a.kv_heads);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, D = (int)a.head_dim;
  const int b = paged::block_find_seq(a.q_start, (int)a.seqs, t, &slot);
  const T *kc = static_cast<const T *>(a.k_cache) + hk * a.k_cache_head;
  const T *vc = static_cast<const T *>(a.v_cache) + hk * a.v_cache_head;
  float q[PER], o[PER], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < D ? paged::to_f32(static_cast<const T *>(a.q)[t * a.q_token + h * a.q_head + d]) * (float)a.scale : 0.f;
    o[i] = 0.f;
  }
  auto visit = [&](const int32_t *pages, int64_t j) {  // key j of a page list
    const int page = pages[j / a.page_size];
    const int64_t s = j % a.page_size;
    const bool ok = paged::page_ok(page, a.pages);
    const T *kr = kc + (ok ? page * a.k_page + s * a.k_slot : 0), *vr = vc + (ok ? page * a.v_page + s * a.v_slot : 0);
    float x = 0.f, v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int d = lane + 32 * i;
      const bool in = ok && d < D;
      x += q[i] * (in ? paged::to_f32(kr[d]) : 0.f);
      v[i] = in ? paged::to_f32(vr[d]) : 0.f;
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
    const float mn = fmaxf(m, x), base = base_of(mn), f = __expf(m - base), p = __expf(x - base);
    m = mn;
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = o[i] * f + p * v[i];
  };
  if (b >= 0) {
    for (int64_t j = warp; j < a.prefix_len; j += WARPS) visit(a.prefix_pages, j);
    const int first = a.q_start ? a.q_start[b] : t, n = a.q_start ? a.q_start[b + 1] - first : 1;
    const int64_t pos = (int64_t)a.kv_len[b] - n + (t - first), end = min(pos + 1, a.table_width * a.page_size);
    const int64_t low = a.window > 0 ? max((int64_t)0, pos - a.window + 1) : 0;
    const int32_t *pages = a.page_table + b * a.table_stride;
    const int64_t head = min(min(a.sinks, low), end);
    for (int64_t j = warp; j < head; j += WARPS) visit(pages, j);
    for (int64_t j = low + warp; j < end; j += WARPS) visit(pages, j);
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 32 * i < D) s_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_m[w]);
  const float base = base_of(M);
  for (int w = 0; w < WARPS; ++w) L += s_l[w] == 0.f ? 0.f : s_l[w] * __expf(s_m[w] - base);
  for (int d = threadIdx.x; d < D; d += WARPS * 32) {
    float x = 0.f;
    for (int w = 0; w < WARPS; ++w) x += s_l[w] == 0.f ? 0.f : s_o[w][d] * __expf(s_m[w] - base);
    static_cast<T *>(a.out)[t * a.out_token + h * a.out_head + d] = paged::from_f32<T>(L == 0.f ? 0.f : x / L);
  }
}

// what a call's sizes must be, without its arrays
int check_sizes(const Args &a) {
  auto bad = [](const char *m) { return fail(NKB_ERR_INVALID, std::string("paged_attention: ") + m); };
  if (int s = paged::check_cache("paged_attention", a.tokens, a.seqs, a.kv_heads, a.head_dim, a.pages, a.page_size,
                                 a.table_width, a.table_stride))
    return s;
  if (!paged::float_dtype(a.dtype))
    return fail(NKB_ERR_UNSUPPORTED, "paged_attention: q, out and caches must be float32, bfloat16 or float16");
  if (a.q_heads < 1 || a.q_heads % a.kv_heads || a.q_heads > 65535) return bad("q_heads must be a multiple of kv_heads");
  if (a.head_dim > MAX_D) return fail(NKB_ERR_UNSUPPORTED, "paged_attention: head_dim above 256");
  if (a.window < 0 || a.sinks < 0 || a.prefix_len < 0) return bad("window, sinks and prefix_len must not be negative");
  if (a.prefix_len > paged::MAX_POSITIONS) return bad("prefix of more than 2^31 - 256 positions");
  if (a.prefix_len && a.window) return fail(NKB_ERR_UNSUPPORTED, "paged_attention: a window over a shared prefix");
  if (!a.q_start && a.tokens != a.seqs) return bad("without q_start there is one token per sequence");
  return NKB_OK;
}

int check_arrays(const Args &a) {
  auto bad = [](const char *m) { return fail(NKB_ERR_INVALID, std::string("paged_attention: ") + m); };
  if (a.tokens && (!a.q || !a.out || !a.kv_len || (a.table_width && !a.page_table) || (a.pages && (!a.k_cache || !a.v_cache))))
    return bad("NULL array");
  if (a.tokens && a.prefix_len && !a.prefix_pages) return bad("a prefix needs its pages");
  if (!std::isfinite(a.scale)) return bad("scale must be finite");
  return NKB_OK;
}

// One new token per sequence of a 16-bit type, rows of whole 16-byte pieces,
// up to 128 dimensions: the split decode kernel.  (By the sizes; an unaligned
// array then takes the form for any layout.)
bool decode_form(const Args &a) {
  return !a.q_start && a.dtype != NKB_F32 && a.head_dim <= 128 && a.seqs * a.q_heads <= INT32_MAX;
}

// The tiles mask a score before it is scaled, and take the largest score as the
// largest scaled one: a scale (in their log2 units, fp32) that is zero, negative or
// subnormal takes the form for any layout, which scales first.
bool tile_scale(const Args &a) { return (float)(a.scale * LOG2E) >= FLT_MIN; }

// Tokens by q_start: the tensor-core tiles, for page sizes that a block of 128
// keys is made of.
bool several_form(const Args &a) { return a.q_start && tile_form(a); }
// A shared prefix: its part on the tiles, the rest by either form.
bool prefix_form(const Args &a) { return a.prefix_len > 0 && tile_form(a) && (a.q_start || decode_form(a)); }

int workspace(const Args &a, int device, size_t *bytes) {
  if (int s = check_sizes(a)) return s;
  if (!a.tokens) *bytes = 0;
  else if (a.prefix_len) *bytes = prefix_form(a) ? prefix_workspace(a, device) : 0;
  else if (decode_form(a)) *bytes = decode_workspace(a, device, false);
  else *bytes = several_form(a) ? tile_workspace(a, device, true, false, false) : 0;
  return NKB_OK;
}

int run(const Args &a, int device, cudaStream_t st) {
  size_t need = 0;
  if (int s = workspace(a, device, &need)) return s;
  if (int s = check_arrays(a)) return s;
  if (a.workspace_bytes < (int64_t)need || (need && !a.workspace))
    return fail(NKB_ERR_INVALID, "paged_attention: workspace of " + std::to_string(a.workspace_bytes) + " bytes, " +
                                     std::to_string(need) + " needed");
  if (reinterpret_cast<uintptr_t>(a.workspace) & 15) return fail(NKB_ERR_INVALID, "paged_attention: unaligned workspace");
  if (a.tokens == 0) return NKB_OK;
  if (a.prefix_len) {
    if (prefix_form(a) && tile_strides(a) && tile_scale(a)) return prefix_run(a, st, device);
  } else if (decode_form(a) && aligned16(a)) {
    single::Params p;
    decode_params(a, device, a.workspace, false, &p);
    return decode_launch(p, st, device, false);
  } else if (several_form(a) && tile_strides(a) && tile_scale(a)) {
    several::Params p;
    tile_params(a, device, a.workspace, true, false, false, &p);
    return tile_launch(p, st, device);
  }
  paged::with_dtype(a.dtype, [&](auto t) {
    attn_any_kernel<decltype(t)><<<dim3((unsigned)a.tokens, (unsigned)a.q_heads), WARPS * 32, 0, st>>>(a);
    return 0;
  });
  return launch_status("paged_attention");
}

// "paged_attention": the pointers of nkb_paged_attention_args that are given;
// ints a mask of them and the struct's integers; floats scale
int check(const Step &s) {
  Args a;
  if (int e = paged::step_args(s, nullptr, 9, 24, "paged_attention", &a)) return e;
  if (int e = check_sizes(a)) return e;
  return check_arrays(a);
}
int launch(const LaunchArgs &l) {
  Args a;
  if (int e = paged::step_args(*l.step, l.ptrs, 9, 24, "paged_attention", &a)) return e;
  return run(a, l.device, l.stream);
}

}  // namespace pattn

NKB_REGISTER_KERNEL("paged_attention", pattn::launch, pattn::check);

}  // namespace nkb

extern "C" int nkb_paged_attention_workspace(const nkb_paged_attention_args *args, size_t *bytes) {
  if (!args || !bytes) return nkb::fail(NKB_ERR_INVALID, "NULL argument");
  int dev = 0;
  cudaGetDevice(&dev);
  return nkb::pattn::workspace(*args, dev, bytes);
}

extern "C" int nkb_paged_attention(const nkb_paged_attention_args *args, void *stream) {
  if (!args) return nkb::fail(NKB_ERR_INVALID, "args is NULL");
  int dev = 0;
  cudaGetDevice(&dev);
  return nkb::pattn::run(*args, dev, static_cast<cudaStream_t>(stream));
}
