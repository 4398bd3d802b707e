// beam.hip — one step of a beam search: of all continuations of a group's beams the best, and the reordered state.
//
//   total[b, v] = scores[b] + logits[b, v] - logsumexp(logits[b, :])      of a beam that goes on
//   total[b, eos] = scores[b], every other -inf                            of a finished beam
//   rank = total / length^penalty, length = the continuation's; the `beams` highest win, ties go to the lowest b * vocab + v.
//
// Within a beam the order of the totals is the order of the logits, so the vocabulary is read once: every wave takes a stretch of a row and gives its
// maximum, its sum of exponentials and its `beams` highest logits; a second kernel joins the sums (in 64 bits) and ranks the few that are left, in 64
// bits as well, so that what lies within a rounding to 32 keeps its order within a beam.  Across beams the log-sum-exps decide: the exponentials
// are 32-bit ones and a lane adds its 32 in 32 bits, which the scan has time for beside its loads.  That is good to 5e-8 as a rule; at worst 31 additions lose 31 2^-24
// and the rounding of an exponent (logit - top) log2 e of up to 17 bits 27 2^-24 of the sum, 2^-18 in all.
#include "common.h"

namespace mmamd {

constexpr int kBeamMost = 32;   // beams of a group
constexpr int kBeamUnit = 2048; // logits of a wave: 32 a lane

struct BeamParams {
  const void* logits;
  const float* scores;
  const int32_t* lengths;
  const uint8_t* finished;
  const int64_t* sequences;
  int64_t ld, eos;
  float* out_scores;
  int32_t *out_lengths, *out_parents;
  uint8_t* out_finished;
  int64_t *out_tokens, *out_sequences;
  float* unit_max;      // workspace, per row and unit
  double* unit_sum;
  uint2* unit_top;      // per row, unit and place: (logit, index), best first; index -1 = none
  int groups, beams, vocab, units, tokens;
  double penalty;
};

// a wave's maximum, in every lane, by data-parallel moves (a shuffle goes through LDS); NaN counts as nothing
__device__ __forceinline__ float dpp_max(float v) {
#define MMAMD_DPP_MAX(ctrl, rows) v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), ctrl, rows, 0xf, false)))
  MMAMD_DPP_MAX(0x111, 0xf);  // row_shr:1, 2, 4, 8: lane 15 of each row of 16 has the row's
  MMAMD_DPP_MAX(0x112, 0xf);
  MMAMD_DPP_MAX(0x114, 0xf);
  MMAMD_DPP_MAX(0x118, 0xf);
  MMAMD_DPP_MAX(0x142, 0xa);  // row_bcast:15 and :31: lane 63 has all
  MMAMD_DPP_MAX(0x143, 0xc);
#undef MMAMD_DPP_MAX
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

__device__ __forceinline__ double dpp_max(double v) {
#define MMAMD_DPP_MAX(ctrl, rows)                                                                                                                     \
  v = fmax(v, __hiloint2double(__builtin_amdgcn_update_dpp(__double2hiint(v), __double2hiint(v), ctrl, rows, 0xf, false),                             \
                               __builtin_amdgcn_update_dpp(__double2loint(v), __double2loint(v), ctrl, rows, 0xf, false)))
  MMAMD_DPP_MAX(0x111, 0xf);
  MMAMD_DPP_MAX(0x112, 0xf);
  MMAMD_DPP_MAX(0x114, 0xf);
  MMAMD_DPP_MAX(0x118, 0xf);
  MMAMD_DPP_MAX(0x142, 0xa);
  MMAMD_DPP_MAX(0x143, 0xc);
#undef MMAMD_DPP_MAX
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), 63), __builtin_amdgcn_readlane(__double2loint(v), 63));
}

// a wave's sum, in every lane
__device__ __forceinline__ double dpp_sum(double v) {
#define MMAMD_DPP_ADD(ctrl, rows)                                                                                                                \
  v += __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), ctrl, rows, 0xf, false),                                              \
                        __builtin_amdgcn_update_dpp(0, __double2loint(v), ctrl, rows, 0xf, false))
  MMAMD_DPP_ADD(0x111, 0xf);
  MMAMD_DPP_ADD(0x112, 0xf);
  MMAMD_DPP_ADD(0x114, 0xf);
  MMAMD_DPP_ADD(0x118, 0xf);
  MMAMD_DPP_ADD(0x142, 0xa);
  MMAMD_DPP_ADD(0x143, 0xc);
#undef MMAMD_DPP_ADD
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), 63), __builtin_amdgcn_readlane(__double2loint(v), 63));
}

template <typename T>
__device__ __forceinline__ void beam_load4(const T* p, bool vec, int left, float (&f)[4]) {
  if (vec && left >= 4) {
    const f32x4 v = load4(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = j < left ? to_f32<T>(p[j]) : -INFINITY;
  }
}

// grid: ceil(units / 4) x rows, one unit a wave.  Of the lanes' maxima the `beams`-th highest is a bound that the unit's `beams` best do not fall below:
// what lies above it (32 values for each of fewer than `beams` lanes, at most, a handful as a rule) and the first of its equals are gathered in LDS,
// where each counts how many are better.  (Taking the best `beams` times over all 32 values of a lane was bound by its compares and shuffles: 39 us for
// 512 rows of 49408, 12 us for 5; this way 19 and 6.)  Bound by HBM: 101 MB in 19 us, 5.3 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void beam_scan_kernel(const BeamParams p) {
  extern __shared__ uint2 lists[];
  const int row = blockIdx.y, unit = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, K = p.beams;
  if (unit >= p.units || p.finished[row] || !(p.scores[row] > -INFINITY)) return;  // nobody reads the units of such a row
  uint2* list = lists + (threadIdx.x >> 6) * 32 * K;
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  const bool vec = (reinterpret_cast<uintptr_t>(x) & (4 * sizeof(T) - 1)) == 0;
  const int base = unit * kBeamUnit + lane * 4;
  float f[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) beam_load4<T>(x + base + i * 256, vec, p.vocab - (base + i * 256), f[i]);
  float mine = -INFINITY;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) mine = fmaxf(mine, f[i][j]);
  const float top = dpp_max(mine);
  // 32 terms a lane in 32 bits, the lanes in 64; the difference first, so that the terms that count are the exact ones.  With no maximum (all -inf) there
  // is no sum; a NaN or +inf makes it NaN.
  float part = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) part += __builtin_amdgcn_exp2f((f[i][j] - top) * 1.4426950408889634f);
  double sum = dpp_sum(top > -INFINITY ? (double)part : 0.0);
  if (__any(!(part == part)) && top > -INFINITY) sum = NAN;
  const int64_t at = (int64_t)row * p.units + unit;
  if (top == -INFINITY) {  // nothing but -inf, or NaN and -inf: told apart here
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) nan |= !(f[i][j] == f[i][j]);
    if (__any(nan)) sum = NAN;
  }
  if (lane == 0) { p.unit_max[at] = top; p.unit_sum[at] = sum; }

  float left = mine, bound = top;
  for (int k = 0; k < K && bound > -INFINITY; ++k) {
    bound = dpp_max(left);
    const unsigned long long who = __ballot(left == bound);
    if (lane == __ffsll(who) - 1) left = -INFINITY;
  }
  int n = 0;  // gathered, the same in every lane
  const unsigned long long below = (1ull << lane) - 1;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned long long who = __ballot(f[i][j] > bound);
      if (who != 0) {
        if (f[i][j] > bound) list[n + __popcll(who & below)] = make_uint2(__float_as_uint(f[i][j]), (uint32_t)(base + i * 256 + j));
        n += __popcll(who);
      }
    }
  if (bound > -INFINITY) {
    const int above = n;
    int equal = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      int before = 0, all = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned long long who = __ballot(f[i][j] == bound);
        before += __popcll(who & below);
        all += __popcll(who);
      }
      if (all != 0 && above + equal < K) {
        int rank = equal + before;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (f[i][j] == bound) {
            if (above + rank < K) list[above + rank] = make_uint2(__float_as_uint(bound), (uint32_t)(base + i * 256 + j));
            ++rank;
          }
      }
      equal += all;
    }
    n = above + equal < K ? above + equal : (above > K ? above : K);
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's list is in LDS
  uint2* out = p.unit_top + at * K;
  for (int e = lane; e < n; e += 64) {
    const uint2 me = list[e];
    const float v = __uint_as_float(me.x);
    int better = 0;
    for (int d = 0; d < n; ++d) {
      const uint2 y = list[d];
      const float w = __uint_as_float(y.x);
      better += w > v || (w == v && y.y < me.y);
    }
    if (better < K) out[better] = me;
  }
  if (lane >= n && lane < K) out[lane] = make_uint2(0xff800000u, 0xffffffffu);  // none
}

// The `beams` best of a row, from the units' lists: each is in order, so the best that is left is at one of their heads.  A lane watches M neighbouring units,
// so that of equal logits the lowest lane's is the lowest word.  stage: the first S of every list, in LDS; the rest is read where it lies.  Lane k gets the k-th.
constexpr int kBeamStage = 256;
// Up to this many beams every pair of a group's continuations is compared at once (beams^4 pairs), beyond it the beams' lists are put in order and merged.  Us a
// call, 25 groups of 49408 words, pairs / merged: 4 beams 16.1 / 17.0, 5: 18.3 / 19.3, 8: 27.1 / 23.8, 9: 33.7 / 25.7.
constexpr int kBeamPairs = 6;
template <int M>
__device__ __forceinline__ int merge_units(const uint2* list, const uint2* stage, int units, int S, int K, int lane, float& mine, uint32_t& word) {
  float hv[M];
  uint32_t hi[M];
  int pos[M];
#pragma unroll
  for (int j = 0; j < M; ++j) {
    const int u = lane * M + j;
    const uint2 e = u < units ? stage[u * S] : make_uint2(0xff800000u, 0xffffffffu);
    hv[j] = __uint_as_float(e.x);
    hi[j] = e.y;
    pos[j] = 0;
  }
  int found = 0;
  for (; found < K; ++found) {
    float bv = hv[0];
    uint32_t bi = hi[0];
    int bj = 0;
#pragma unroll
    for (int j = 1; j < M; ++j)
      if (hv[j] > bv) { bv = hv[j]; bi = hi[j]; bj = j; }
    const float best = dpp_max(bv);
    if (!(best > -INFINITY)) break;
    const int win = __ffsll((unsigned long long)__ballot(bv == best)) - 1;
    const uint32_t low = (uint32_t)__builtin_amdgcn_readlane((int)bi, win);
    if (lane == found) { mine = best; word = low; }
    if (lane == win) {
#pragma unroll
      for (int j = 0; j < M; ++j)
        if (j == bj) {
          const int at = ++pos[j], u = lane * M + j;
          uint2 e = make_uint2(0xff800000u, 0xffffffffu);
          if (at < S) e = stage[u * S + at];
          else if (at < K) e = list[(int64_t)u * K + at];
          hv[j] = __uint_as_float(e.x);
          hi[j] = e.y;
        }
    }
  }
  return found;
}

// One workgroup per group.  A wave per beam joins the sums and merges the units' lists into the beam's `beams` best; then the beams are merged (or compared
// in pairs).  Bound by its chain of dependent steps -- 7 us for up to 5 beams, 11 for 9, 44 for 32, of which the units' lists take half -- so everything that can be
// loaded is loaded at once: a row that was not scanned has whatever lay in the workspace, and does not use it.  (Looking through all candidates for every place,
// and beams^4 pairs, took a call of one group from 15 us with 5 beams to 62 with 12, 119 with 16 and 1114 with 32; now 22, 27 and 56.)
__global__ __launch_bounds__(1024) void beam_join_kernel(const BeamParams p) {
  __shared__ double total[kBeamMost * kBeamMost];  // of the continuations of all beams: beam * beams + place
  __shared__ double rank[kBeamMost * kBeamMost];
  __shared__ uint32_t token[kBeamMost * kBeamMost];
  __shared__ int better[kBeamPairs * kBeamPairs], place[kBeamMost], len[kBeamMost];
  __shared__ bool fin[kBeamMost];
  __shared__ uint2 stages[16][kBeamStage];
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, K = p.beams;
  uint2* const stage = stages[wave];
  const int S = p.units * K <= kBeamStage ? K : kBeamStage / p.units;  // (0 for more units than a merge takes)
  for (int b = wave; b < K; b += blockDim.x >> 6) {
    const int row = g * K + b;
    const uint2* list = p.unit_top + (int64_t)row * p.units * K;
    const float* um = p.unit_max + (int64_t)row * p.units;
    const double* us = p.unit_sum + (int64_t)row * p.units;
    uint2 head[kBeamStage / 64];
#pragma unroll
    for (int j = 0; j < kBeamStage / 64; ++j) {
      const int e = lane + j * 64;
      head[j] = list[e < p.units * S ? (S == K ? e : e / S * K + e % S) : 0];
    }
    const float m0 = lane < p.units ? um[lane] : -INFINITY;
    const double s0 = lane < p.units ? us[lane] : 0.0;
    const bool done = p.finished[row] != 0;
    const double score = (double)p.scores[row];
    const int after = p.lengths[row] + (done ? 0 : 1);
#pragma unroll
    for (int j = 0; j < kBeamStage / 64; ++j) stage[lane + j * 64] = head[j];
    double lse = NAN;
    if (!done && score > -INFINITY) {
      float top = m0;
      for (int u = lane + 64; u < p.units; u += 64) top = fmaxf(top, um[u]);
      top = dpp_max(top);
      double sum = m0 > -INFINITY ? s0 * exp((double)m0 - (double)top) : s0;
      for (int u = lane + 64; u < p.units; u += 64) sum += um[u] > -INFINITY ? us[u] * exp((double)um[u] - (double)top) : us[u];
      lse = (double)top + log(dpp_sum(sum));
    }
    double mark = -INFINITY;       // lane k's continuation, k < K: its total and its word
    uint32_t word = 0xffffffffu;
    if (lse > -INFINITY && lse < INFINITY) {
      float mine = -INFINITY;
      int found = 0;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's stage is in LDS
      if (p.units <= 64) {
        found = merge_units<1>(list, stage, p.units, S, K, lane, mine, word);
      } else if (p.units <= kBeamStage) {
        found = merge_units<kBeamStage / 64>(list, stage, p.units, S, K, lane, mine, word);
      } else {                                            // a vocabulary of more than 524288: every place looks through all lists
        float v0 = INFINITY;
        uint32_t i0 = 0;
        for (; found < K; ++found) {
          float bv = -INFINITY;
          uint32_t bi = 0xffffffffu;
          for (int c = lane; c < p.units * K; c += 64) {
            const uint2 e = list[c];
            const float v = __uint_as_float(e.x);
            if ((v < v0 || (v == v0 && e.y > i0)) && (v > bv || (v == bv && e.y < bi))) { bv = v; bi = e.y; }
          }
          const float best = dpp_max(bv);
          if (!(best > -INFINITY)) break;
          uint32_t low = bv == best ? bi : 0xffffffffu;
#pragma unroll
          for (int o = 32; o > 0; o >>= 1) { const uint32_t y = __shfl_xor(low, o); low = y < low ? y : low; }
          v0 = best;
          i0 = low;
          if (lane == found) { mine = best; word = low; }
        }
      }
      if (lane < found) mark = score + ((double)mine - lse);
      if (found < K) {                                    // all finite ones are listed: the first words that are not, at -inf
        if (lane < found) token[b * K + lane] = word;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        uint32_t t = 0;
        for (int k = found; k < K; ++k, ++t) {            // (every lane alike)
          for (int d = 0; d < found; ++d)
            if (token[b * K + d] == t) { ++t; d = -1; }
          if (lane == k) word = t < (uint32_t)p.vocab ? t : 0xffffffffu;
        }
      }
    } else if (lane < K) {
      // a finished beam goes on as it is; every other continuation of it, and all of a dead beam, tie at -inf: the first ones of them
      const int eos = (int)p.eos;
      const bool alive = done && score > -INFINITY;
      const int t = !alive ? lane : lane == 0 ? eos : (lane - 1 < eos ? lane - 1 : lane);
      if (alive && lane == 0) mark = score;
      word = t < p.vocab ? (uint32_t)t : 0xffffffffu;
    }
    if (lane < K) {
      total[b * K + lane] = mark;
      token[b * K + lane] = word;
    }
    if (lane == 0) { fin[b] = done; len[b] = after; }
  }
  __syncthreads();
  // a thread per continuation: its rank, and its place among its beam's -- a rank may be a tie where the logits were none, and the lower word comes first then
  const bool mine = tid < K * K;                          // (the workgroup has as many threads)
  const int first = tid / K * K;                          // of the beam
  double mark = 0.0, r = 0.0;
  uint32_t word = 0xffffffffu;
  if (mine) {
    mark = total[tid];
    word = token[tid];
    const double base = (double)(len[tid / K] > 1 ? len[tid / K] : 1);
    r = p.penalty == 0.0 ? mark : mark / (p.penalty == 1.0 ? base : pow(base, p.penalty));
    if (!(r == r)) r = -INFINITY;                         // (-inf over a power that overflows; every pair has to have an order)
    rank[tid] = r;
    if (K <= kBeamPairs) better[tid] = 0;
  }
  __syncthreads();
  if (K <= kBeamPairs) {                                  // every pair of continuations is compared by a thread of its own
    const int all = K * K;
    for (int x = tid; x < all * all; x += blockDim.x) {
      const int c = x / all, d = x - c * all;
      const double a = rank[c], q = rank[d];
      if (token[d] != 0xffffffffu && (q > a || (q == a && (d / K < c / K || (d / K == c / K && token[d] < token[c]))))) atomicAdd(&better[c], 1);
    }
    __syncthreads();
    if (mine && word != 0xffffffffu && better[tid] < K) place[better[tid]] = tid;
  } else {
    int at = 0;
    if (mine) {
#pragma unroll 4
      for (int d = first; d < first + K; ++d) {
        const double q = rank[d];
        const uint32_t y = token[d];                      // none (a vocabulary smaller than the beams): behind the others
        at += word == 0xffffffffu ? y != word || d < tid : y != 0xffffffffu && (q > r || (q == r && y < word));
      }
    }
    __syncthreads();
    if (mine) {
      total[first + at] = mark;
      rank[first + at] = r;
      token[first + at] = word;
    }
    __syncthreads();
    if (wave == 0) {                                      // lane b watches beam b; of equal ranks the lowest beam's comes first
      int c = lane * K;
      bool some = lane < K && token[c] != 0xffffffffu;
      double v = some ? rank[c] : -INFINITY;
      for (int k = 0; k < K; ++k) {
        const double best = dpp_max(v);
        const unsigned long long who = __ballot(some && v == best);
        if (lane == __ffsll(who) - 1) {
          place[k] = c++;
          some = c < (lane + 1) * K && token[c] != 0xffffffffu;
          v = some ? rank[c] : -INFINITY;
        }
      }
    }
  }
  __syncthreads();
  for (int k = tid; k < K; k += blockDim.x) {
    const int c = place[k], b = c / K, to = g * K + k;
    p.out_scores[to] = (float)total[c];
    p.out_lengths[to] = len[b];
    p.out_finished[to] = fin[b] || token[c] == (uint32_t)p.eos;
    p.out_tokens[to] = token[c];
    p.out_parents[to] = g * K + b;
  }
  if (p.out_sequences == nullptr) return;
  for (int k = wave; k < K; k += blockDim.x >> 6) {
    const int c = place[k], b = c / K, at = fin[b] ? -1 : len[b] - 1;
    const int64_t* from = p.sequences + (int64_t)(g * K + b) * p.tokens;
    int64_t* to = p.out_sequences + (int64_t)(g * K + k) * p.tokens;
    for (int t = lane; t < p.tokens; t += 64) to[t] = t == at ? (int64_t)token[c] : from[t];
  }
}

}  // namespace mmamd

using namespace mmamd;

static int beam_check(const char* who, int groups, int beams, int vocab) {
  MMAMD_CHECK_ARG(groups >= 0 && beams >= 1 && vocab >= 1, MMAMD_E_BADARG, "%s: groups %d, beams %d, vocabulary %d", who, groups, beams, vocab);
  MMAMD_CHECK_ARG(beams <= kBeamMost && (int64_t)groups * beams <= 65535 && vocab <= 0x7fffffff - 65536, MMAMD_E_UNSUPPORTED,
                  "%s: %d groups of %d beams (at most %d beams, 65535 in all)", who, groups, beams, kBeamMost);
  return 0;
}
static int beam_units(int vocab) { return (vocab + kBeamUnit - 1) / kBeamUnit; }

extern "C" int64_t mmamd_beam_search_workspace(int groups, int beams, int vocab) {
  if (int rc = beam_check("mmamd_beam_search_workspace", groups, beams, vocab)) return rc;
  return (int64_t)groups * beams * beam_units(vocab) * (16 + 8 * beams);
}

extern "C" int mmamd_beam_search_step(const void* logits, int dtype, int64_t ld, const float* scores, const int32_t* lengths, const uint8_t* finished, const int64_t* sequences,
                                      int tokens, int64_t eos, double length_penalty, int groups, int beams, int vocab, float* out_scores, int32_t* out_lengths, uint8_t* out_finished,
                                      int64_t* out_tokens, int32_t* out_parents, int64_t* out_sequences, void* workspace, int64_t workspace_bytes, mmamd_stream_t stream) {
  if (int rc = beam_check("mmamd_beam_search_step", groups, beams, vocab)) return rc;
  if (groups == 0) return 0;
  MMAMD_CHECK_ARG(dtype == MMAMD_F32 || dtype == MMAMD_BF16, MMAMD_E_UNSUPPORTED, "mmamd_beam_search_step: dtype code %d (fp32 / bf16 only)", dtype);
  MMAMD_CHECK_ARG(logits && scores && lengths && finished && out_scores && out_lengths && out_finished && out_tokens && out_parents && workspace && (sequences == nullptr) == (out_sequences == nullptr),
                  MMAMD_E_BADARG, "mmamd_beam_search_step: null argument");
  MMAMD_CHECK_ARG(ld >= 0 && tokens >= 0 && eos >= 0 && eos < vocab && length_penalty - length_penalty == 0.0, MMAMD_E_BADARG,
                  "mmamd_beam_search_step: ld %lld, tokens %d, eos %lld of a vocabulary of %d, length penalty %f", (long long)ld, tokens, (long long)eos, vocab, length_penalty);
  const int64_t need = mmamd_beam_search_workspace(groups, beams, vocab);
  MMAMD_CHECK_ARG(workspace_bytes >= need && aligned16(workspace), MMAMD_E_BADARG, "mmamd_beam_search_step: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  BeamParams p;
  p.logits = logits; p.scores = scores; p.lengths = lengths; p.finished = finished; p.sequences = sequences;
  p.ld = ld; p.eos = eos;
  p.out_scores = out_scores; p.out_lengths = out_lengths; p.out_finished = out_finished; p.out_tokens = out_tokens; p.out_parents = out_parents; p.out_sequences = out_sequences;
  p.groups = groups; p.beams = beams; p.vocab = vocab; p.units = beam_units(vocab); p.tokens = tokens; p.penalty = length_penalty;
  const int64_t n = (int64_t)groups * beams * p.units;
  p.unit_top = reinterpret_cast<uint2*>(workspace);
  p.unit_sum = reinterpret_cast<double*>(p.unit_top + n * beams);
  p.unit_max = reinterpret_cast<float*>(p.unit_sum + n);
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((p.units + 3) / 4, groups * beams);
  const int lds = 4 * 32 * beams * 8;  // at most 32 values of `beams` lanes in the list of each wave: 32 KiB
  if (dtype == MMAMD_F32) beam_scan_kernel<float><<<grid, 256, lds, st>>>(p);
  else beam_scan_kernel<bf16><<<grid, 256, lds, st>>>(p);
  if (int rc = launch_status("beam_search_step scan")) return rc;
  beam_join_kernel<<<groups, 64 * (beams < 8 ? 8 : beams < 16 ? beams : 16), 0, st>>>(p);
  return launch_status("beam_search_step");
}
