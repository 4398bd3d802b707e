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

// LDS transpose read: within each 16-lane group, lane i points at 4 contiguous 16-bit values -- row i >> 2, columns 4 (i & 3) .. + 3 of a [4][16] block --
// and receives column i of the block.
typedef __attribute__((ext_vector_type(4))) short s16x4;
__device__ __forceinline__ s16x4 lds_columns(const bf16* at) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at); }

template <typename T>
__device__ __forceinline__ f32x4 mma16(const uint4& a, const uint4& b, f32x4 c);  // c += a b over the 4 pieces of 16 bytes that 4 lanes hold of a row
template <>
__device__ __forceinline__ f32x4 mma16<bf16>(const uint4& a, const uint4& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma16<float>(const uint4& a, const uint4& b, f32x4 c) {
  const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
  return c;
}

template <bool STREAM>
__device__ __forceinline__ uint4 load_piece(const char* at) {
  if constexpr (STREAM) return load_past(at);
  else return *reinterpret_cast<const uint4*>(at);
}

// the maximum over the four lanes l, l + 16, l + 32, l + 48, in each of them (a shuffle would go through LDS)
__device__ __forceinline__ float across_quarters_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// One workgroup: up to 16 query heads of one key head of one row over one split of the row's tokens, so that the cache is requested once for every 16 query heads
// of a key head (a group of 33: three times), and once for every row that reads a page (beams that share an image's states: 32 x 5 rows over 256 tokens, 12 x 64,
// request 126 MB of 25 MB, 14.0 us a call).  The four waves take the split's tiles (32 tokens in bf16, 16 in fp32) in turn, each with its own running maximum, sum and output:
//   scores [token, head] = K . q: the tile's keys go from memory to the registers of a 16 x 16 product as they lie (lane = token, 4 lanes share a row);
//   out [dim, head] += V^T . weights: the values go through LDS for their columns, the weights are where the first product left them.
// A pass over a tile ends with the loads of the next one in flight, and the page numbers of the one after.  fp32 runs on the fp32 matrix instruction.
// bf16 weights are used as two bf16 parts (2^-18 of a weight is lost): in one part they would lose as much as the output's own rounding.
// Measured, us a call and TB/s of the keys and values: 4 rows of 65536 tokens, 8 x 128, 4 query heads each: 166, 6.5 (a large copy: 4.9); 61 rows of 0 .. 8192
// tokens, 12 x 64: 67, 4.8 -- what is missing are the first loads of each workgroup and the join; one row of 40 tokens: 5.0 (4.2 in a graph), latency.  Two waves a SIMD
// are enough (with 96 and 128 wide heads; bounds of three or four spill there: 308 and 453 us on the first of these).
// GROUPS: 16 tokens that begin at a multiple of 16 lie in one page (the page size is a multiple of 16), so their addresses are one scalar and a
// constant lane offset; otherwise every lane finds the page of one token and the others' come by shuffles.
template <typename T, int D, bool STREAM, bool GROUPS>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(const PagedAttnParams p) {
  constexpr int TOK = sizeof(T) == 2 ? 32 : 16;      // tokens of a tile
  constexpr int NT = TOK / 16;
  constexpr int PIECES = D * (int)sizeof(T) / 16;    // 16-byte pieces of a row
  constexpr int KP = PIECES / 4, VP = TOK * PIECES / 64;
  constexpr int VROW = D + 16 / (int)sizeof(T);      // row of the values in LDS: the odd 16 bytes spread 16 rows over the banks
  constexpr int ND = D / 16;
  constexpr int RROW = D + 4;
  constexpr int VBYTES = TOK * VROW * (int)sizeof(T), RBYTES = 16 * RROW * 4;
  __shared__ __attribute__((aligned(16))) char smem[4 * (VBYTES > RBYTES ? VBYTES : RBYTES)];
  __shared__ float red_m[4][16], red_l[4][16];

  const int row = blockIdx.z, kvh = blockIdx.y / p.sub, sg = blockIdx.y - kvh * p.sub, split = blockIdx.x;
  int pos;
  const int n = row_tokens(p, row, pos);
  const int chunk = row_chunk(p, n);
  const int begin = split * chunk, end = (begin + chunk < n) ? begin + chunk : n;
  if (begin >= n && split != 0) return;              // (split 0 of an empty row writes its zeros)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, quarter = lane >> 4;
  const int h0 = kvh * p.group + sg * 16;
  const int nh = (p.group - sg * 16) < 16 ? (p.group - sg * 16) : 16;
  T* vs = reinterpret_cast<T*>(smem + wave * VBYTES);

  uint4 qf[KP];
  {
    const T* qp = reinterpret_cast<const T*>(p.q) + row * p.q_row + (h0 + (l15 < nh ? l15 : 0)) * p.q_head;
#pragma unroll
    for (int i = 0; i < KP; ++i) qf[i] = reinterpret_cast<const uint4*>(qp)[i * 4 + quarter];
  }
  const int32_t* table = p.table + row * p.table_row;
  char* const keys = reinterpret_cast<char*>(p.keys) + kvh * p.key_head * (int64_t)sizeof(T);
  char* const values = reinterpret_cast<char*>(p.values) + kvh * p.value_head * (int64_t)sizeof(T);
  const char* const knew = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.k) + row * p.k_row + kvh * p.k_head);
  const char* const vnew = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.v) + row * p.v_row + kvh * p.v_head);

  constexpr int VG = VP / NT;                        // pieces of values per lane and 16 tokens
  uint4 kr[NT][KP], vr[VP];
  uint32_t okmask = 0;                               // which tokens of the loaded tile take part
  constexpr uint32_t ALL = TOK == 32 ? 0xffffffffu : 0xffffu;
  auto value_place = [&](int i, int& tok, int& x) {  // piece i of this lane: its token in the tile, its place in the token's row
    const int piece = i % VG * 64 + lane;
    tok = i / VG * 16 + piece / PIECES;
    x = piece % PIECES;
  };
  // The tile's page numbers, raw: looking at one here would wait for it and thereby for the tile that was just requested.  For groups they are scalar loads,
  // which count apart from the others (the table is not written while this runs: the address space says so).
  struct Ids { int id[GROUPS ? NT : 1]; };
  typedef const __attribute__((address_space(4))) int32_t* const_ptr;
  auto page_of = [&](int t0) {
    Ids r;
    if constexpr (GROUPS) {
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const int t = t0 + u * 16;
        r.id[u] = ((const_ptr)(uintptr_t)table)[div_by(p.page, (uint32_t)(t < end ? t : end - 1))];
      }
    } else {
      const int t = t0 + (lane & (TOK - 1));
      r.id[0] = table[div_by(p.page, (uint32_t)(t < end ? t : end - 1))];
    }
    return r;
  };
  const uint32_t klane = (uint32_t)(l15 * p.key_token * (int64_t)sizeof(T)) + quarter * 16;  // (GROUPS only, where it fits)
  auto load_tile = [&](int t0, const Ids& ids) {
    if constexpr (GROUPS) {
      okmask = 0;
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const int t = t0 + u * 16, off = t - (int)(div_by(p.page, (uint32_t)t) * p.page.d), left = end - t;
        const bool inside = (uint32_t)ids.id[u] < (uint32_t)p.pages && left > 0;
        if (inside) okmask |= (left >= 16 ? 0xffffu : (1u << left) - 1u) << (u * 16);
        const int64_t pg = inside ? ids.id[u] : 0;           // a place that holds no token is read as page 0, which exists, and not used
        const char* kb = keys + (pg * p.key_page + off * p.key_token) * (int64_t)sizeof(T);
        const char* vb = values + (pg * p.value_page + off * p.value_token) * (int64_t)sizeof(T);
#pragma unroll
        for (int i = 0; i < KP; ++i) kr[u][i] = load_piece<STREAM>(kb + klane + i * 64);
#pragma unroll
        for (int i = 0; i < VG; ++i) {
          int tok, x;
          value_place(i, tok, x);
          vr[u * VG + i] = load_piece<STREAM>(vb + (uint32_t)(tok * p.value_token * (int64_t)sizeof(T)) + x * 16);
        }
      }
    } else {
      const int t = t0 + (lane & (TOK - 1)), id = ids.id[0];
      const bool inside = (uint32_t)id < (uint32_t)p.pages && t < end;
      okmask = (uint32_t)__ballot(inside && lane < TOK);
      const int off = t - (int)(div_by(p.page, (uint32_t)t) * p.page.d);
      const int64_t pg = inside ? id : 0;
      const int64_t ko = (pg * p.key_page + off * p.key_token) * (int64_t)sizeof(T), vo = (pg * p.value_page + off * p.value_token) * (int64_t)sizeof(T);
      const int klo = (int)ko, khi = (int)(ko >> 32), vlo = (int)vo, vhi = (int)(vo >> 32);
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const int64_t o = (int64_t)(((uint64_t)(uint32_t)__shfl(khi, u * 16 + l15) << 32) | (uint32_t)__shfl(klo, u * 16 + l15));
#pragma unroll
        for (int i = 0; i < KP; ++i) kr[u][i] = load_piece<STREAM>(keys + o + (i * 4 + quarter) * 16);
      }
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        int tok, x;
        value_place(i, tok, x);
        const int64_t o = (int64_t)(((uint64_t)(uint32_t)__shfl(vhi, tok) << 32) | (uint32_t)__shfl(vlo, tok));
        vr[i] = load_piece<STREAM>(values + o + x * 16);
      }
    }
    if (pos >= t0 && pos < t0 + TOK && (okmask >> (pos - t0) & 1u)) {  // the new token is not in its place yet
#pragma unroll
      for (int u = 0; u < NT; ++u)
        if (t0 + u * 16 + l15 == pos) {
#pragma unroll
          for (int i = 0; i < KP; ++i) kr[u][i] = *reinterpret_cast<const uint4*>(knew + (i * 4 + quarter) * 16);
        }
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        int tok, x;
        value_place(i, tok, x);
        if (t0 + tok == pos) vr[i] = *reinterpret_cast<const uint4*>(vnew + x * 16);
      }
    }
  };

  float m = -3.402823466e38f, l = 0.f;
  f32x4 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};

  int t0 = begin + wave * TOK;
  Ids ids;
  if (t0 < end) {
    ids = page_of(t0);
    load_tile(t0, ids);
    ids = page_of(t0 + 4 * TOK);
  }
  for (; t0 < end; t0 += 4 * TOK) {
    const uint32_t ok = okmask;
    if (pos >= t0 && pos < t0 + TOK && sg == 0 && (ok >> (pos - t0) & 1u)) {  // the new token into its place
      const int slot = (int)div_by(p.page, (uint32_t)pos), off = pos - slot * (int)p.page.d;
      const int64_t pg = table[slot];
      char* kd = keys + (pg * p.key_page + off * p.key_token) * (int64_t)sizeof(T);
      char* vd = values + (pg * p.value_page + off * p.value_token) * (int64_t)sizeof(T);
#pragma unroll
      for (int u = 0; u < NT; ++u)
        if (t0 + u * 16 + l15 == pos) {
#pragma unroll
          for (int i = 0; i < KP; ++i) *reinterpret_cast<uint4*>(kd + (i * 4 + quarter) * 16) = kr[u][i];
        }
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        int tok, x;
        value_place(i, tok, x);
        if (t0 + tok == pos) *reinterpret_cast<uint4*>(vd + x * 16) = vr[i];
      }
    }
    f32x4 s[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KP; ++i) s[u] = mma16<T>(kr[u][i], qf[i], s[u]);
    }
    const bool whole = ok == ALL;
    if (!whole) {                                      // what lies where no token is may be anything, NaN too
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        int tok, x;
        value_place(i, tok, x);
        if (!(ok >> tok & 1u)) vr[i] = make_uint4(0, 0, 0, 0);
      }
      asm volatile("");                                // (a branch, not a select in every tile)
    }
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      int tok, x;
      value_place(i, tok, x);
      *reinterpret_cast<uint4*>(vs + tok * VROW + x * (16 / (int)sizeof(T))) = vr[i];
    }
    if (t0 + 4 * TOK < end) {
      load_tile(t0 + 4 * TOK, ids);
      ids = page_of(t0 + 8 * TOK);
    }
    // weights: this lane has head l15 and the tokens u * 16 + 4 quarter + i
    float top = m;
#pragma unroll
    for (int u = 0; u < NT; ++u) s[u] *= p.scale_log2e;
    if (!whole) {
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(ok >> (u * 16 + quarter * 4 + i) & 1u)) s[u][i] = -INFINITY;
      asm volatile("");
    }
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, s[u][i]);
    top = across_quarters_max(top);
    if (__any(top > m)) {                              // (as a rule the maximum is found early)
      const float fac = __builtin_amdgcn_exp2f(m - top);
      m = top;
      l *= fac;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= fac;
    }
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[u][i] = __builtin_amdgcn_exp2f(s[u][i] - top);
        l += s[u][i];
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave's values are in LDS
    if constexpr (sizeof(T) == 2) {
      bf16x8 hi, lo;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          hi[u * 4 + i] = (bf16)s[u][i];
          lo[u * 4 + i] = (bf16)(s[u][i] - (float)hi[u * 4 + i]);
        }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const bf16* at = reinterpret_cast<const bf16*>(vs) + (quarter * 4 + (l15 >> 2)) * VROW + d * 16 + (l15 & 3) * 4;
        const s16x4 a0 = lds_columns(at), a1 = lds_columns(at + 16 * VROW);
        typedef __attribute__((ext_vector_type(8))) short s16x8;
        const bf16x8 a = __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, hi, o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, lo, o[d], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(reinterpret_cast<const float*>(vs)[(quarter * 4 + i) * VROW + d * 16 + l15], s[0][i], o[d], 0, 0, 0);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // ... and read, before the next tile's overwrite them
  }
  // join the four waves
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  __syncthreads();
  float* const red = reinterpret_cast<float*>(smem);
  if (l15 < nh) {
    float* r = red + (wave * 16 + l15) * RROW + quarter * 4;
#pragma unroll
    for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4*>(r + d * 16) = o[d];
    if (quarter == 0) { red_m[wave][l15] = m; red_l[wave][l15] = l; }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nh * D; i += 256) {
    const int g = i / D, d = i - g * D;
    float top = red_m[0][g];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, red_m[w][g]);
    float ls = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float fac = __builtin_amdgcn_exp2f(red_m[w][g] - top);
      ls = fmaf(red_l[w][g], fac, ls);
      v = fmaf(red[(w * 16 + g) * RROW + d], fac, v);
    }
    const int64_t rh = (int64_t)row * p.heads + h0 + g;
    if (n <= chunk) {  // one split holds the whole row
      reinterpret_cast<T*>(p.out)[rh * D + d] = (T)(ls == 0.f ? 0.f : v / ls);
    } else {
      const int64_t at = rh * p.splits + split;
      p.ws[at * D + d] = v;
      if (d == 0) reinterpret_cast<float2*>(p.ws + (int64_t)p.rows * p.heads * p.splits * D)[at] = make_float2(top, ls);
    }
  }
}

// Joins the splits of a (row, head): o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  The statistics of all splits first, one a thread; then the
// outputs, each group of D threads every NG-th split, whose loads do not wait for one another.  The first of them are requested before the statistics are joined: 61
// rows of up to 8192 tokens 67.15 -> 66.65 us a call; the kernel takes 4 to 5, a chain of loads.
constexpr int kSplitsMost = 256;
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedAttnParams p) {
  constexpr int NG = 256 / D;
  __shared__ float w[kSplitsMost], part[NG][D], red[4], sums[4];
  const int h = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int pos;
  const int n = row_tokens(p, row, pos);
  const int64_t rh = (int64_t)row * p.heads + h;
  float2 ml = tid < p.splits ? reinterpret_cast<const float2*>(p.ws + (int64_t)p.rows * p.heads * p.splits * D)[rh * p.splits + tid] : make_float2(0.f, 0.f);
  const int chunk = row_chunk(p, n);
  if (n <= chunk) return;                               // a single split has written its output
  const int used = (n + chunk - 1) / chunk;
  if (tid >= used) ml = make_float2(-3.402823466e38f, 0.f);  // (what nobody wrote)
  const int g = tid / D, d = tid - g * D;
  const float* const o = p.ws + rh * p.splits * D + d;
  constexpr int AHEAD = 8;                              // outputs that are requested before the statistics are there
  float ahead[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int s = g + k * NG;
    ahead[k] = o[(int64_t)(g < NG && s < used ? s : 0) * D];
  }
  float top = wave_max(ml.x);
  if (lane == 0) red[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float f = __builtin_amdgcn_exp2f(ml.x - top);
  w[tid] = tid < used ? f : 0.f;
  const float ls = wave_sum(ml.y * f);
  if (lane == 0) sums[wave] = ls;
  __syncthreads();
  if (g < NG) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (g + k * NG < used) v = fmaf(w[g + k * NG], ahead[k], v);
#pragma unroll 8
    for (int s = g + AHEAD * NG; s < used; s += NG) v = fmaf(w[s], o[(int64_t)s * D], v);
    part[g][d] = v;
  }
  __syncthreads();
  if (tid < D) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < NG; ++k) v += part[k][tid];
    const float total = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    reinterpret_cast<T*>(p.out)[rh * D + tid] = (T)(total == 0.f ? 0.f : v / total);
  }
}

// Splits of a row, from what the host knows: the workgroups without splits (rows x key heads x 16s of a group) and the capacity of the page table (the lengths
// are on the device; a kernel that finds a row shorter cuts it into fewer, of 128 tokens at least).  A split costs a second kernel, about 3 us.
// Us a call, 12 heads of 64 in bf16, one split / more:
//   one row        256 tokens 4.9 / 6.7, 512: 6.5 / 6.7, 1024: 9.6 / 7.0              -> one up to 64 KiB of keys a head
//   32 rows        1024 tokens 18.4 / 21.5, 2048: 31.1 / 35.4, 4096: 73.7 / 74.8    -> one up to 256 KiB if there is a workgroup for every CU;
//   61 rows, mixed up to 8192     stretches of 1024 tokens 66.9, of 2048: 69.9      -> beyond that, stretches of 1024: long rows must not end last
//   5 rows         4096 tokens, 18 splits 16.9, 33: 16.6, 9: 18.7                     -> few rows: 1024 workgroups, stretches of 2048 at most
static int paged_splits(int64_t wgs, int64_t capacity, int row_bytes) {
  const int64_t whole = 65536 / row_bytes;
  const bool full = wgs >= kChipCUs;
  if (capacity <= (full ? 4 * whole : whole)) return 1;
  int64_t s = full ? (capacity + 1023) / 1024 : (capacity + 2047) / 2048;
  const int64_t fill = (1024 + wgs - 1) / wgs;
  if (!full && s < fill) s = fill;
  const int64_t most = (capacity + 127) / 128, grid = 16384 / wgs;
  if (s > most) s = most;
  if (s > grid) s = grid;
  if (s > kSplitsMost) s = kSplitsMost;
  return s < 1 ? 1 : (int)s;
}
static int paged_splits(const mmamd_paged_cache* c, int rows, int heads) {
  const int64_t sub = (heads / c->kv_heads + 15) / 16;
  return paged_splits((int64_t)rows * c->kv_heads * sub, (int64_t)c->slots * c->page_size, c->dim * (c->dtype == MMAMD_F32 ? 4 : 2));
}

// A pool of this size or less is read through the caches as usual, a larger one past them: two of the 256 MB that the last cache holds, since a decoder reads its pool
// again and again, and rows that share pages read them from there.  Us a call, as usual / past them: 1.07 GB 188 / 166; 322 MB, none of it cached, 66.5 / 62.9; 50 MB
// whose pages eight rows share 33 / 50; 25 MB shared by five 14.0 / 18.3.
constexpr int64_t kStreamBytes = 512ll << 20;

template <typename T, int D>
static int launch_paged_attn(PagedAttnParams& p, hipStream_t st) {
  p.sub = (p.group + 15) / 16;
  p.min_chunk = 128;
  const dim3 grid(p.splits, p.kv_heads * p.sub, p.rows);
  const int64_t pool = 2ll * p.pages * p.kv_heads * p.page.d * D * (int64_t)sizeof(T);
  const bool groups = p.page.d % 16 == 0 && p.key_token * (int64_t)sizeof(T) < 1 << 26 && p.value_token * (int64_t)sizeof(T) < 1 << 26;  // (lane offsets of 32 bits)
  const bool past = pool > kStreamBytes;
  if (groups && past) paged_attn_kernel<T, D, true, true><<<grid, 256, 0, st>>>(p);
  else if (groups) paged_attn_kernel<T, D, false, true><<<grid, 256, 0, st>>>(p);
  else if (past) paged_attn_kernel<T, D, true, false><<<grid, 256, 0, st>>>(p);
  else paged_attn_kernel<T, D, false, false><<<grid, 256, 0, st>>>(p);
  if (int rc = launch_status("paged_attention")) return rc;
  if (p.splits > 1) {
    paged_join_kernel<T, D><<<dim3(p.heads, p.rows), 256, 0, st>>>(p);
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

// Four 16-byte pieces a thread, all loaded before the first is stored; consecutive threads walk the pieces of a head, the heads and the tokens, so both sides
// see whole rows.
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendParams p) {
  const int row = blockIdx.y;
  int count = p.counts != nullptr ? p.counts[row] : p.tokens;
  count = count < p.tokens ? count : p.tokens;
  const int64_t start = p.start[row];
  const uint32_t total = count > 0 ? (uint32_t)count * p.per_token.d : 0u;
  const uint32_t first = blockIdx.x * 1024u + threadIdx.x;
  uint4 piece[4];
  char* to[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t i = first + k * 256u;
    to[k] = nullptr;
    if (i >= total) continue;
    const uint32_t j = div_by(p.per_token, i), x = i - j * p.per_token.d;   // token, place within it
    const uint32_t hv = div_by(p.per_head, x), at = (x - hv * p.per_head.d) * 16u;
    const bool val = hv >= (uint32_t)p.kv_heads;
    const int h = (int)(val ? hv - p.kv_heads : hv);
    const int64_t t = start + j;
    if (t < 0 || t >= (int64_t)p.slots * p.page.d) continue;
    const uint32_t slot = div_by(p.page, (uint32_t)t), off = (uint32_t)t - slot * p.page.d;
    const int id = p.table[row * p.table_row + slot];
    if ((uint32_t)id >= (uint32_t)p.pages) continue;
    const char* src = val ? reinterpret_cast<const char*>(p.v) + row * p.v_row + j * p.v_token + h * p.v_head
                          : reinterpret_cast<const char*>(p.k) + row * p.k_row + j * p.k_token + h * p.k_head;
    to[k] = (val ? reinterpret_cast<char*>(p.values) + id * p.value_page + h * p.value_head + off * p.value_token
                 : reinterpret_cast<char*>(p.keys) + id * p.key_page + h * p.key_head + off * p.key_token) + at;
    piece[k] = *reinterpret_cast<const uint4*>(src + at);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (to[k] != nullptr) store_past(to[k], piece[k]);
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
  const int s = paged_splits(c, rows, heads);
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
  p.splits = paged_splits(c, rows, heads);
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
