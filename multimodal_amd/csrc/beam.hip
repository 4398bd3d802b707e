// beam.hip — one step of a beam search: of all continuations of a group's beams the best, and the reordered state.
//
//   total[b, v] = scores[b] + logits[b, v] - logsumexp(logits[b, :])      of a beam that goes on
//   total[b, eos] = scores[b], every other -inf                            of a finished beam
//   rank = total / length^penalty, length = the continuation's; the `beams` highest win, ties go to the lowest b * vocab + v.
//
// Within a beam the order of the totals is the order of the logits, so the vocabulary is read once: every wave takes a stretch of a row and gives its
// maximum, its sum of exponentials and its `beams` highest logits; a second kernel joins the sums (in 64 bits) and ranks the few that are left, in 64
// bits as well, since two continuations may lie as near to each other as a rounding to 32.
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
  uint2* unit_top;      // per row, unit and place: (order key, index); key 0 = none
  int groups, beams, vocab, units, tokens;
  double penalty;
};

// floats in the order of unsigned integers; NaN counts as -inf here (a row that holds one is dead by its sum)
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  const uint32_t k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return x == x ? k : 0x007fffffu;  // the key of -inf
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

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

// grid: ceil(units / 4) x rows, one unit a wave
template <typename T>
__global__ __launch_bounds__(256) void beam_scan_kernel(const BeamParams p) {
  const int row = blockIdx.y, unit = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (unit >= p.units || p.finished[row] || !(p.scores[row] > -INFINITY)) return;  // nobody reads the units of such a row
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  const bool vec = (reinterpret_cast<uintptr_t>(x) & (4 * sizeof(T) - 1)) == 0;
  const int base = unit * kBeamUnit + lane * 4;
  float f[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) beam_load4<T>(x + base + i * 256, vec, p.vocab - (base + i * 256), f[i]);
  float top = -INFINITY;
  uint32_t key[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      top = fmaxf(top, f[i][j]);
      key[i][j] = base + i * 256 + j < p.vocab ? order_key(f[i][j]) : 0u;
    }
  top = wave_max(top);
  // 32 terms a lane in 32 bits, the lanes in 64.  With no maximum (all -inf) there is no sum either; a NaN or +inf makes it NaN.
  float part = 0.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (base + i * 256 + j < p.vocab) nan |= !(f[i][j] < INFINITY);
      part += top > -INFINITY ? expf(f[i][j] - top) : 0.f;
    }
  double sum = (double)part;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (__any(nan)) sum = NAN;
  const int64_t at = (int64_t)row * p.units + unit;
  if (lane == 0) { p.unit_max[at] = top; p.unit_sum[at] = sum; }
  for (int k = 0; k < p.beams; ++k) {
    uint32_t best = 0;
    int where = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (key[i][j] > best) { best = key[i][j]; where = i * 4 + j; }
    uint32_t all = best;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { const uint32_t y = __shfl_xor(all, o); all = y > all ? y : all; }
    const int idx = base + (where >> 2) * 256 + (where & 3);
    int low = best == all && all != 0 ? idx : 0x7fffffff;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { const int y = __shfl_xor(low, o); low = y < low ? y : low; }
    if (lane == 0) p.unit_top[at * p.beams + k] = make_uint2(all, (uint32_t)low);
    if (all != 0 && low == idx) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (where == i * 4 + j) key[i][j] = 0;
    }
  }
}

// is (key, index) of one candidate of a beam behind another's: lower, or as high and further back
__device__ __forceinline__ bool behind(uint32_t k, uint32_t i, uint32_t k0, uint32_t i0) { return k < k0 || (k == k0 && i > i0); }

// One workgroup per group.  A wave per beam joins the sums and merges the units' lists into the beam's `beams` best; the continuations of all beams then
// count how many are better than they, which is their place.
__global__ __launch_bounds__(256) void beam_join_kernel(const BeamParams p) {
  __shared__ double rank[kBeamMost * kBeamMost];
  __shared__ float total[kBeamMost * kBeamMost];
  __shared__ uint32_t token[kBeamMost * kBeamMost];
  __shared__ int place[kBeamMost];
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, K = p.beams;
  for (int b = wave; b < K; b += 4) {
    const int row = g * K + b;
    const bool fin = p.finished[row] != 0;
    const double score = (double)p.scores[row];
    double lse = NAN;
    if (!fin && score > -INFINITY) {
      const float* um = p.unit_max + (int64_t)row * p.units;
      const double* us = p.unit_sum + (int64_t)row * p.units;
      float top = -INFINITY;
      for (int u = lane; u < p.units; u += 64) top = fmaxf(top, um[u]);
      top = wave_max(top);
      double sum = 0.0;
      for (int u = lane; u < p.units; u += 64) sum += um[u] > -INFINITY ? us[u] * exp((double)um[u] - (double)top) : us[u];
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
      lse = (double)top + log(sum);
    }
    const int len = p.lengths[row] + (fin ? 0 : 1);
    const double div = pow((double)(len > 1 ? len : 1), p.penalty);
    if (lse > -INFINITY && lse < INFINITY) {
      const uint2* list = p.unit_top + (int64_t)row * p.units * K;
      uint32_t k0 = 0xffffffffu, i0 = 0;
      for (int k = 0; k < K; ++k) {
        uint32_t bk = 0, bi = 0xffffffffu;
        for (int c = lane; c < p.units * K; c += 64) {
          const uint2 e = list[c];
          if (e.x != 0 && behind(e.x, e.y, k0, i0) && (e.x > bk || (e.x == bk && e.y < bi))) { bk = e.x; bi = e.y; }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
          const uint32_t yk = __shfl_xor(bk, o), yi = __shfl_xor(bi, o);
          if (yk > bk || (yk == bk && yi < bi)) { bk = yk; bi = yi; }
        }
        if (lane == 0) {
          const float logit = key_value(bk);
          const double t = bk != 0 && logit > -INFINITY ? score + ((double)logit - lse) : -INFINITY;
          rank[b * K + k] = t / div;
          total[b * K + k] = (float)t;
          token[b * K + k] = bk != 0 ? bi : 0xffffffffu;  // (a vocabulary smaller than the beams)
        }
        k0 = bk; i0 = bi;
      }
    } else if (lane < K) {
      // a finished beam goes on as it is; every other continuation of it, and all of a dead beam, tie at -inf: the first ones of them
      const int eos = (int)p.eos;
      const bool alive = fin && score > -INFINITY;
      const int t = !alive ? lane : lane == 0 ? eos : (lane - 1 < eos ? lane - 1 : lane);
      const double own = alive && lane == 0 ? score : -INFINITY;
      rank[b * K + lane] = own / div;
      token[b * K + lane] = t < p.vocab ? (uint32_t)t : 0xffffffffu;
      total[b * K + lane] = (float)own;
    }
  }
  __syncthreads();
  for (int c = tid; c < K * K; c += 256) {
    if (token[c] == 0xffffffffu) continue;
    const double r = rank[c];
    const int64_t flat = (int64_t)(c / K) * p.vocab + token[c];
    int better = 0;
    for (int d = 0; d < K * K; ++d)
      better += token[d] != 0xffffffffu && (rank[d] > r || (rank[d] == r && (int64_t)(d / K) * p.vocab + token[d] < flat));
    if (better < K) place[better] = c;
  }
  __syncthreads();
  for (int k = tid; k < K; k += 256) {
    const int c = place[k], b = c / K, row = g * K + b, to = g * K + k;
    const bool fin = p.finished[row] != 0;
    const int len = p.lengths[row] + (fin ? 0 : 1);
    p.out_scores[to] = total[c];
    p.out_lengths[to] = len;
    p.out_finished[to] = fin || token[c] == (uint32_t)p.eos;
    p.out_tokens[to] = token[c];
    p.out_parents[to] = row;
  }
  if (p.out_sequences == nullptr) return;
  for (int64_t i = tid; i < (int64_t)K * p.tokens; i += 256) {
    const int k = (int)(i / p.tokens), t = (int)(i - (int64_t)k * p.tokens);
    const int c = place[k], row = g * K + c / K;
    const bool put = p.finished[row] == 0 && t == p.lengths[row];
    p.out_sequences[(int64_t)g * K * p.tokens + i] = put ? (int64_t)token[c] : p.sequences[(int64_t)row * p.tokens + t];
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
  MMAMD_CHECK_ARG(ld >= 0 && tokens >= 0 && eos >= 0 && eos < vocab && length_penalty == length_penalty, MMAMD_E_BADARG,
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
  if (dtype == MMAMD_F32) beam_scan_kernel<float><<<grid, 256, 0, st>>>(p);
  else beam_scan_kernel<bf16><<<grid, 256, 0, st>>>(p);
  if (int rc = launch_status("beam_search_step scan")) return rc;
  beam_join_kernel<<<groups, 256, 0, st>>>(p);
  return launch_status("beam_search_step");
}
