// paged_attention.hip — attention of one new token per sequence over a key-value cache that lives in pages, and the write of prompts into the pages.
//
//   o[r, h] = sum_t softmax_t(scale q[r, h] . K[r, t, h / G]) V[r, t, h / G]        t < n_r,  G = heads / kv_heads
//
// token t of row r lies in page page_table[r, t / page] at place t % page.  A page number outside the pool holds no tokens: its positions take no part.
// With k and v given the row's new token is first stored at position lengths[r] and takes part.
//
// What bounds it: the cache is read once, 2 n_r kv_heads dim values, for 4 n_r heads dim flop -- G flop per byte in bf16, HBM.
#include "paged.h"

namespace mmamd {

struct PagedAttnParams {
  const void *q, *k, *v;
  void *keys, *values;
  const int32_t *table, *lengths;
  void* out;
  float* ws;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, key_page, key_head, key_token, value_page, value_head, value_token, table_row;
  int rows, heads, kv_heads, group, sub, pages, slots, splits, min_chunk;
  FastDiv page;
  float scale_log2e;
};

// 16 bytes of T as floats
template <typename T>
struct Vec16;
template <>
struct Vec16<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
};
template <>
struct Vec16<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
};

// the tokens [begin, end) of a row that split s of it takes; chunks of at least min_chunk tokens, so that a short row is not cut up.  Every kernel
// that needs to know which splits of a row hold anything asks here.
__device__ __forceinline__ int row_chunk(const PagedAttnParams& p, int n) {
  const int c = (n + p.splits - 1) / p.splits;
  return c < p.min_chunk ? p.min_chunk : ((c + 63) & ~63);
}
// visible tokens of a row: the cached ones and, with k given, the new one where it has a place
__device__ __forceinline__ int row_tokens(const PagedAttnParams& p, int row, int& pos) {
  const int cap = p.slots * (int)p.page.d;
  const int len = p.lengths[row];
  pos = -1;
  if (p.k != nullptr && len >= 0 && len < cap) pos = len;
  return pos >= 0 ? len + 1 : clamp_int(len, 0, cap);
}

// One workgroup: GT query heads of one key head of one row over one split of the row's tokens.  Four lanes share a token (each a quarter of its
// dims, in 16-byte pieces), a wave has 16 tokens in flight per step and U steps at once; every lane group keeps the running maximum, sum and output
// of its own tokens in fp32, joined by shuffles at the end, the four waves through LDS, the splits by paged_join_kernel.
template <typename T, int D, int GT, int U>
__global__ __launch_bounds__(256) void paged_attn_kernel(const PagedAttnParams p) {
  constexpr int EV = Vec16<T>::N;               // values per 16 bytes
  constexpr int NV = D / (4 * EV);              // 16-byte pieces per lane and token
  constexpr int DL = NV * EV;                   // values per lane and token
  const int row = blockIdx.z, kvh = blockIdx.y / p.sub, sg = blockIdx.y - kvh * p.sub, split = blockIdx.x;
  int pos;
  const int n = row_tokens(p, row, pos);
  const int chunk = row_chunk(p, n);
  const int begin = split * chunk, end = (begin + chunk < n) ? begin + chunk : n;
  if (begin >= n && !(split == 0)) return;      // (split 0 of an empty row writes its zeros)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 3, quad = lane >> 2;
  const int h0 = kvh * p.group + sg * GT;
  const int nh = (p.group - sg * GT) < GT ? (p.group - sg * GT) : GT;

  float q[GT][DL];
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    const T* qp = reinterpret_cast<const T*>(p.q) + row * p.q_row + (h0 + (g < nh ? g : 0)) * p.q_head;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[EV];
      Vec16<T>::unpack(*reinterpret_cast<const uint4*>(qp + (i * 4 + c) * EV), f);
#pragma unroll
      for (int e = 0; e < EV; ++e) q[g][i * EV + e] = f[e] * p.scale_log2e;
    }
  }
  float m[GT], l[GT], o[GT][DL];
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    m[g] = -3.402823466e38f;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < DL; ++e) o[g][e] = 0.f;
  }
  const int32_t* table = p.table + row * p.table_row;
  const T* keys = reinterpret_cast<const T*>(p.keys) + kvh * p.key_head;
  const T* values = reinterpret_cast<const T*>(p.values) + kvh * p.value_head;
  const T* knew = reinterpret_cast<const T*>(p.k) + row * p.k_row + kvh * p.k_head;
  const T* vnew = reinterpret_cast<const T*>(p.v) + row * p.v_row + kvh * p.v_head;

  for (int t0 = begin + wave * 16 * U; t0 < end; t0 += 4 * 16 * U) {
    uint4 kr[U][NV], vr[U][NV];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * 16 + quad;
      const int tc = t < end ? t : end - 1;                     // loads never leave the row
      const int slot = (int)div_by(p.page, (uint32_t)tc), off = tc - slot * (int)p.page.d;
      const int id = table[slot];
      const bool inside = (uint32_t)id < (uint32_t)p.pages;
      ok[u] = inside && t < end;
      const int64_t pg = inside ? id : 0;
      T* kp = const_cast<T*>(keys) + pg * p.key_page + off * p.key_token;
      T* vp = const_cast<T*>(values) + pg * p.value_page + off * p.value_token;
      const bool fresh = t == pos;
      const T* ks = fresh ? knew : kp;
      const T* vs = fresh ? vnew : vp;
#pragma unroll
      for (int i = 0; i < NV; ++i) kr[u][i] = *reinterpret_cast<const uint4*>(ks + (i * 4 + c) * EV);
#pragma unroll
      for (int i = 0; i < NV; ++i) vr[u][i] = *reinterpret_cast<const uint4*>(vs + (i * 4 + c) * EV);
      if (fresh && ok[u] && sg == 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          *reinterpret_cast<uint4*>(kp + (i * 4 + c) * EV) = kr[u][i];
          *reinterpret_cast<uint4*>(vp + (i * 4 + c) * EV) = vr[u][i];
        }
      }
      if (!ok[u]) {  // what lies in a place that holds no token may be anything, NaN too
#pragma unroll
        for (int i = 0; i < NV; ++i) vr[u][i] = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      float s[U], top = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float f[EV];
          Vec16<T>::unpack(kr[u][i], f);
#pragma unroll
          for (int e = 0; e < EV; ++e) a = fmaf(q[g][i * EV + e], f[e], a);
        }
        a += __shfl_xor(a, 1);
        a += __shfl_xor(a, 2);
        s[u] = ok[u] ? a : -INFINITY;
        top = fmaxf(top, s[u]);
      }
      const float fac = __builtin_amdgcn_exp2f(m[g] - top);
      m[g] = top;
      l[g] *= fac;
#pragma unroll
      for (int e = 0; e < DL; ++e) o[g][e] *= fac;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float w = __builtin_amdgcn_exp2f(s[u] - top);
        l[g] += w;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float f[EV];
          Vec16<T>::unpack(vr[u][i], f);
#pragma unroll
          for (int e = 0; e < EV; ++e) o[g][i * EV + e] = fmaf(w, f[e], o[g][i * EV + e]);
        }
      }
    }
  }
  // join the 16 lane groups of the wave, then the four waves
  __shared__ float red[4][GT][D + 2];
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    float top = m[g];
#pragma unroll
    for (int x = 4; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float fac = __builtin_amdgcn_exp2f(m[g] - top);
    float ls = l[g] * fac;
#pragma unroll
    for (int x = 4; x < 64; x <<= 1) ls += __shfl_xor(ls, x);
#pragma unroll
    for (int e = 0; e < DL; ++e) {
      float v = o[g][e] * fac;
#pragma unroll
      for (int x = 4; x < 64; x <<= 1) v += __shfl_xor(v, x);
      if (quad == 0) red[wave][g][((e / EV) * 4 + c) * EV + e % EV] = v;
    }
    if (lane == 0) { red[wave][g][D] = top; red[wave][g][D + 1] = ls; }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nh * D; i += 256) {
    const int g = i / D, d = i - g * D;
    float top = red[0][g][D];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, red[w][g][D]);
    float ls = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float fac = __builtin_amdgcn_exp2f(red[w][g][D] - top);
      ls = fmaf(red[w][g][D + 1], fac, ls);
      v = fmaf(red[w][g][d], fac, v);
    }
    const int64_t rh = (int64_t)row * p.heads + h0 + g;
    if (p.splits == 1) {
      reinterpret_cast<T*>(p.out)[rh * D + d] = (T)(ls == 0.f ? 0.f : v / ls);
    } else {
      float* w = p.ws + (rh * p.splits + split) * (D + 2);
      w[d] = v;
      if (d == 0) { w[D] = top; w[D + 1] = ls; }
    }
  }
}

// Joins the splits of a (row, head): o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.
template <typename T, int D>
__global__ __launch_bounds__(D) void paged_join_kernel(const PagedAttnParams p) {
  const int h = blockIdx.x, row = blockIdx.y, d = threadIdx.x;
  int pos;
  const int n = row_tokens(p, row, pos);
  const int chunk = row_chunk(p, n);
  const int used = n > 0 ? (n + chunk - 1) / chunk : 1;
  const int64_t rh = (int64_t)row * p.heads + h;
  const float* w = p.ws + rh * p.splits * (D + 2);
  float top = -3.402823466e38f, ls = 0.f, v = 0.f;
  for (int s = 0; s < used; ++s, w += D + 2) {
    const float ms = w[D], nt = fmaxf(top, ms);
    const float fa = __builtin_amdgcn_exp2f(top - nt), fb = __builtin_amdgcn_exp2f(ms - nt);
    ls = ls * fa + w[D + 1] * fb;
    v = v * fa + w[d] * fb;
    top = nt;
  }
  reinterpret_cast<T*>(p.out)[rh * D + d] = (T)(ls == 0.f ? 0.f : v / ls);
}

// Splits of a row, from what the host knows: the rows, heads and the capacity of the page table (the lengths are on the device).
static int paged_splits(int rows, int heads, int kv_heads, int64_t capacity) {
  const int64_t wgs = (int64_t)rows * kv_heads;
  int64_t s = (capacity + 1023) / 1024;
  const int64_t fill = (2048 + wgs - 1) / wgs;
  if (s < fill) s = fill;
  const int64_t most = (capacity + 127) / 128;
  if (s > most) s = most;
  const int64_t grid = 16384 / wgs;
  if (s > grid) s = grid;
  return s < 1 ? 1 : (int)s;
}

template <typename T, int D>
static int launch_paged_attn(PagedAttnParams& p, hipStream_t st) {
  constexpr int GT = 2;
  const int gt = p.group == 1 ? 1 : GT;
  p.sub = (p.group + gt - 1) / gt;
  p.min_chunk = 128;
  const dim3 grid(p.splits, p.kv_heads * p.sub, p.rows);
  if (gt == 1) paged_attn_kernel<T, D, 1, 2><<<grid, 256, 0, st>>>(p);
  else paged_attn_kernel<T, D, GT, 2><<<grid, 256, 0, st>>>(p);
  if (int rc = launch_status("paged_attention")) return rc;
  if (p.splits > 1) {
    paged_join_kernel<T, D><<<dim3(p.heads, p.rows), D, 0, st>>>(p);
    return launch_status("paged_attention join");
  }
  return 0;
}

template <typename T>
static int launch_paged_attn(PagedAttnParams& p, int dim, hipStream_t st) {
  switch (dim) {
    case 64: return launch_paged_attn<T, 64>(p, st);
    case 96: return launch_paged_attn<T, 96>(p, st);
    default: return launch_paged_attn<T, 128>(p, st);
  }
}

struct PagedAppendParams {
  const void *k, *v;
  void *keys, *values;
  const int32_t *table, *start, *counts;
  int64_t k_row, k_token, k_head, v_row, v_token, v_head, key_page, key_head, key_token, value_page, value_head, value_token, table_row;
  int tokens, kv_heads, pieces, pages, slots;
  FastDiv page, per_token, per_head;
};

// One 16-byte piece per thread and step; consecutive threads walk the pieces of a head, the heads and the tokens, so both sides see whole rows.
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendParams p) {
  const int row = blockIdx.y;
  int count = p.counts != nullptr ? p.counts[row] : p.tokens;
  count = count < p.tokens ? count : p.tokens;
  const int64_t start = p.start[row];
  const uint32_t total = count > 0 ? (uint32_t)count * p.per_token.d : 0u;
  for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < total; i += gridDim.x * 256u) {
    const uint32_t j = div_by(p.per_token, i), x = i - j * p.per_token.d;   // token, place within it
    const uint32_t hv = div_by(p.per_head, x), piece = x - hv * p.per_head.d;
    const bool val = hv >= (uint32_t)p.kv_heads;
    const int h = (int)(val ? hv - p.kv_heads : hv);
    const int64_t t = start + j;
    if (t < 0 || t >= (int64_t)p.slots * p.page.d) continue;
    const uint32_t slot = div_by(p.page, (uint32_t)t), off = (uint32_t)t - slot * p.page.d;
    const int id = p.table[row * p.table_row + slot];
    if ((uint32_t)id >= (uint32_t)p.pages) continue;
    const char* src = val ? reinterpret_cast<const char*>(p.v) + row * p.v_row + j * p.v_token + h * p.v_head
                          : reinterpret_cast<const char*>(p.k) + row * p.k_row + j * p.k_token + h * p.k_head;
    char* dst = val ? reinterpret_cast<char*>(p.values) + id * p.value_page + h * p.value_head + off * p.value_token
                    : reinterpret_cast<char*>(p.keys) + id * p.key_page + h * p.key_head + off * p.key_token;
    *reinterpret_cast<uint4*>(dst + piece * 16) = *reinterpret_cast<const uint4*>(src + piece * 16);
  }
}

static bool good_stride(int64_t s, int size) { return s >= 0 && (s * size) % 16 == 0; }

// the checks that both entry points make of the pages and the table
static int check_pages(const char* who, const mmamd_paged_cache* c) {
  MMAMD_CHECK_ARG(c != nullptr, MMAMD_E_BADARG, "%s: null cache", who);
  MMAMD_CHECK_ARG(c->key_pages != nullptr && c->value_pages != nullptr && c->page_table != nullptr, MMAMD_E_BADARG, "%s: null pages or table", who);
  MMAMD_CHECK_ARG(c->dtype == MMAMD_F32 || c->dtype == MMAMD_BF16, MMAMD_E_UNSUPPORTED, "%s: dtype code %d (fp32 / bf16 only)", who, c->dtype);
  MMAMD_CHECK_ARG(c->pages >= 1 && c->page_size >= 1 && c->slots >= 1 && c->kv_heads >= 1, MMAMD_E_BADARG, "%s: pages %d, page size %d, slots %d, kv_heads %d",
                  who, c->pages, c->page_size, c->slots, c->kv_heads);
  MMAMD_CHECK_ARG((int64_t)c->slots * c->page_size <= 1 << 30, MMAMD_E_UNSUPPORTED, "%s: %d slots of %d tokens pass 2^30", who, c->slots, c->page_size);
  MMAMD_CHECK_ARG(c->dim == 64 || c->dim == 96 || c->dim == 128, MMAMD_E_UNSUPPORTED, "%s: head width %d (64, 96, 128 only)", who, c->dim);
  const int size = c->dtype == MMAMD_F32 ? 4 : 2;
  MMAMD_CHECK_ARG(aligned16(c->key_pages) && aligned16(c->value_pages) && good_stride(c->key_page_stride, size) && good_stride(c->key_head_stride, size) &&
                      good_stride(c->key_token_stride, size) && good_stride(c->value_page_stride, size) && good_stride(c->value_head_stride, size) &&
                      good_stride(c->value_token_stride, size),
                  MMAMD_E_ALIGN, "%s: pages must be 16-byte aligned, with strides of whole 16-byte pieces", who);
  return 0;
}

}  // namespace mmamd

using namespace mmamd;

extern "C" int64_t mmamd_paged_attention_workspace(const mmamd_paged_cache* c, int rows, int heads) {
  if (int rc = check_pages("mmamd_paged_attention_workspace", c)) return rc;
  MMAMD_CHECK_ARG(rows >= 0 && heads >= 1 && heads % c->kv_heads == 0, MMAMD_E_BADARG, "mmamd_paged_attention_workspace: rows %d, heads %d, kv_heads %d", rows, heads, c->kv_heads);
  if (rows == 0) return 0;
  const int s = paged_splits(rows, heads, c->kv_heads, (int64_t)c->slots * c->page_size);
  return s == 1 ? 0 : (int64_t)rows * heads * s * (c->dim + 2) * 4;
}

extern "C" int mmamd_paged_attention(const mmamd_paged_cache* c, const int32_t* lengths, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row,
                                     int64_t k_head, const void* v, int64_t v_row, int64_t v_head, void* out, int rows, int heads, float scale, void* workspace,
                                     int64_t workspace_bytes, mmamd_stream_t stream) {
  if (int rc = check_pages("mmamd_paged_attention", c)) return rc;
  MMAMD_CHECK_ARG(rows >= 0 && heads >= 1 && heads % c->kv_heads == 0, MMAMD_E_BADARG, "mmamd_paged_attention: rows %d, heads %d, kv_heads %d", rows, heads, c->kv_heads);
  if (rows == 0) return 0;
  MMAMD_CHECK_ARG(rows <= 65535 && heads <= 65535, MMAMD_E_UNSUPPORTED, "mmamd_paged_attention: %d rows, %d heads (at most 65535)", rows, heads);
  MMAMD_CHECK_ARG(lengths != nullptr && q != nullptr && out != nullptr && (k == nullptr) == (v == nullptr), MMAMD_E_BADARG, "mmamd_paged_attention: null lengths, q, out, or one of k and v");
  const int size = c->dtype == MMAMD_F32 ? 4 : 2;
  MMAMD_CHECK_ARG(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && good_stride(q_row, size) && good_stride(q_head, size) &&
                      (k == nullptr || (good_stride(k_row, size) && good_stride(k_head, size) && good_stride(v_row, size) && good_stride(v_head, size))),
                  MMAMD_E_ALIGN, "mmamd_paged_attention: q, k, v, out must be 16-byte aligned, with strides of whole 16-byte pieces");
  PagedAttnParams p;
  p.q = q; p.k = k; p.v = v; p.keys = c->key_pages; p.values = c->value_pages; p.table = c->page_table; p.lengths = lengths; p.out = out;
  p.ws = reinterpret_cast<float*>(workspace);
  p.q_row = q_row; p.q_head = q_head; p.k_row = k_row; p.k_head = k_head; p.v_row = v_row; p.v_head = v_head;
  p.key_page = c->key_page_stride; p.key_head = c->key_head_stride; p.key_token = c->key_token_stride;
  p.value_page = c->value_page_stride; p.value_head = c->value_head_stride; p.value_token = c->value_token_stride;
  p.table_row = c->table_row_stride;
  p.rows = rows; p.heads = heads; p.kv_heads = c->kv_heads; p.group = heads / c->kv_heads; p.pages = c->pages; p.slots = c->slots;
  p.page = fast_div((uint32_t)c->page_size);
  p.scale_log2e = scale * 1.4426950408889634f;
  p.splits = paged_splits(rows, heads, c->kv_heads, (int64_t)c->slots * c->page_size);
  if (p.splits > 1) {
    const int64_t need = (int64_t)rows * heads * p.splits * (c->dim + 2) * 4;
    MMAMD_CHECK_ARG(workspace != nullptr && workspace_bytes >= need && aligned16(workspace), MMAMD_E_BADARG, "mmamd_paged_attention: workspace of %lld bytes, %lld needed",
                    (long long)workspace_bytes, (long long)need);
  }
  return c->dtype == MMAMD_F32 ? launch_paged_attn<float>(p, c->dim, (hipStream_t)stream) : launch_paged_attn<bf16>(p, c->dim, (hipStream_t)stream);
}

extern "C" int mmamd_paged_append(const mmamd_paged_cache* c, const void* k, int64_t k_row, int64_t k_token, int64_t k_head, const void* v, int64_t v_row, int64_t v_token,
                                  int64_t v_head, const int32_t* start, const int32_t* counts, int rows, int tokens, mmamd_stream_t stream) {
  if (int rc = check_pages("mmamd_paged_append", c)) return rc;
  MMAMD_CHECK_ARG(rows >= 0 && tokens >= 0, MMAMD_E_BADARG, "mmamd_paged_append: rows %d, tokens %d", rows, tokens);
  if (rows == 0 || tokens == 0) return 0;
  MMAMD_CHECK_ARG(k != nullptr && v != nullptr && start != nullptr, MMAMD_E_BADARG, "mmamd_paged_append: null k, v or start");
  const int size = c->dtype == MMAMD_F32 ? 4 : 2;
  MMAMD_CHECK_ARG(aligned16(k) && aligned16(v) && good_stride(k_row, size) && good_stride(k_token, size) && good_stride(k_head, size) && good_stride(v_row, size) &&
                      good_stride(v_token, size) && good_stride(v_head, size),
                  MMAMD_E_ALIGN, "mmamd_paged_append: k and v must be 16-byte aligned, with strides of whole 16-byte pieces");
  PagedAppendParams p;
  p.k = k; p.v = v; p.keys = c->key_pages; p.values = c->value_pages; p.table = c->page_table; p.start = start; p.counts = counts;
  p.k_row = k_row * size; p.k_token = k_token * size; p.k_head = k_head * size; p.v_row = v_row * size; p.v_token = v_token * size; p.v_head = v_head * size;
  p.key_page = c->key_page_stride * size; p.key_head = c->key_head_stride * size; p.key_token = c->key_token_stride * size;
  p.value_page = c->value_page_stride * size; p.value_head = c->value_head_stride * size; p.value_token = c->value_token_stride * size;
  p.table_row = c->table_row_stride;
  p.tokens = tokens; p.kv_heads = c->kv_heads; p.pages = c->pages; p.slots = c->slots;
  p.pieces = c->dim * size / 16;
  const int64_t per_token = 2ll * c->kv_heads * p.pieces;
  MMAMD_CHECK_ARG(rows <= 65535 && per_token * tokens <= 0x7fffffffll, MMAMD_E_UNSUPPORTED, "mmamd_paged_append: %d rows of %d tokens are too many for one call", rows, tokens);
  p.page = fast_div((uint32_t)c->page_size);
  p.per_token = fast_div((uint32_t)per_token);
  p.per_head = fast_div((uint32_t)p.pieces);
  int64_t blocks = (per_token * tokens + 1023) / 1024;  // four pieces a thread
  paged_append_kernel<<<dim3((unsigned)blocks, rows), 256, 0, (hipStream_t)stream>>>(p);
  return launch_status("paged_append");
}
