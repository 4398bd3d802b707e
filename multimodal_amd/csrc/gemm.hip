// gemm.hip — bf16 "NT" GEMM with fused epilogues on the gfx950 matrix cores.
//
//   C[M,N] = act(A[M,K] . W[N,K]^T + bias[N]) (+ residual[M,N])        A, W bf16; accumulate fp32
//
// This one kernel family is ~96 % of the hot path's FLOPs: packed QKV in-projection, attention
// out-projection (+residual), MLP up (+QuickGELU) and down (+residual), and the patch-embedding
// conv expressed as a GEMM.  Both operands are K-contiguous (torch Linear weight layout), so both
// MFMA operand fragments are 16-byte contiguous LDS reads.
//
// Structure (CDNA4-first, not a CUDA tiling):
//   * v_mfma_f32_32x32x16_bf16, operands SWAPPED: the MFMA "A" operand is the W tile (rows = n) and the
//     "B" operand is the activation tile (rows = m), so D[n][m]: each lane owns ONE output row m and
//     4 consecutive columns n per accumulator group -> bias is a float4, bf16 results pack to 8 bytes
//     and, after one v_permlane32_swap per dword, to one 16-byte store per lane (guide T21).
//   * global -> LDS by LDS-DMA (global_load_lds_dwordx4, 1 KiB per wave-instruction, no VGPR round
//     trip).  The DMA destination is lane-linear, so the bank swizzle is applied to the per-lane
//     SOURCE address and undone on the ds_read_b128 side (guide rule 21).  Swizzle: a tile row is
//     128 B (BK = 64 bf16); two rows share a 256-byte bank row of 16 slots; slot' = slot ^ (bankrow & 15)
//     -> every 16-lane ds_read_b128 group hits 16 distinct slots (conflict-free).
//   * 2-stage LDS ring, ONE barrier per K-tile: the DMA for tile k+1 is issued right after the barrier
//     that retires tile k-1's reads, and is only waited for (vmcnt(0)) at the next barrier, a full
//     compute phase later.
//   * XCD-aware bijective block remap: consecutive tile ids land on ONE XCD so the blocks sharing an
//     activation row-panel / the weight matrix hit the same 4 MiB L2.
#include <type_traits>

#include "common.h"

namespace mmamd {

// cache-policy bits of the fp32 epilogue's buffer loads / stores (gfx94x: 1 = sc0, 2 = nt, 16 = sc1); build-time A/B only
#ifndef MMAMD_EPI_LD_AUX
#define MMAMD_EPI_LD_AUX 0
#endif
#ifndef MMAMD_EPI_WIN
#define MMAMD_EPI_WIN 1
#endif
#ifndef MMAMD_EPI_ST_AUX
#define MMAMD_EPI_ST_AUX 16  // sc1: written through, not kept in the XCD's L2 (r06 A/B: the step -0.8 % against plain stores)
#endif

typedef uint32_t __attribute__((address_space(3))) * lds_u32p;
typedef const uint32_t __attribute__((address_space(1))) * glb_u32p;
typedef __attribute__((ext_vector_type(4))) int int32x4;

// LDS-DMA through a buffer descriptor: per-lane 32-bit byte offset (constant over the K loop) + a SCALAR K offset.
// The 64-bit-vaddr form (global_load_lds v[a:a+1], off) needs one v_lshl_add_u64 per piece; measured
// (tools/microbench/mfma_dma_mix.hip) that VALU traffic beside a busy matrix pipe cuts the DMA stream of a CU from
// 57 to 21 B/clk and was the reason every schedule of this kernel stalled at ~40 % MFMA utilisation.  The SRD /
// saddr forms need no VALU at all and run at the full 57 B/clk next to full-rate MFMAs.
__device__ void llvm_amdgcn_raw_buffer_load_lds(int32x4 rsrc, lds_u32p lds_ptr, int size, int voffset, int soffset,
                                                int offset, int aux) __asm("llvm.amdgcn.raw.buffer.load.lds");

__device__ __forceinline__ int32x4 make_srd(const void* base, uint32_t bytes) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  int32x4 r;
  r[0] = (int)(uint32_t)(p & 0xffffffffu);
  r[1] = (int)(uint32_t)((p >> 32) & 0xffffu);  // stride 0 (raw buffer)
  r[2] = (int)bytes;                              // num_records in bytes: reads past the end return 0
  r[3] = 0x00020000;
  return r;
}

struct GemmArgs {
  const bf16* A;
  const bf16* W;
  const float* bias;
  const void* R;
  void* C;
  int M, N, K;
  int lda, ldw, ldr, ldc;
  int act;
  int tiles_n;
  int res_mode;             // 0: C += R;  1 / 2: C *= QuickGELU'(R) / GELU'(R) (backward of the MLP: R = saved pre-activation, bf16)
  int kt_chunk;             // split-K (weight gradients): K-tiles (of 64) per split, blockIdx.y = split; 0 = no split
  long long c_split_stride; // elements between the partial outputs of consecutive splits
  int split_flat;           // split-K with the split index folded into blockIdx.x (1-D grid of tiles * splits, split-major): 0 = blockIdx.y
  void* C2;                 // training forward of the MLP: second bf16 output act2(bf16(C)) next to the pre-activation C (NULL = none)
  int ldc2, act2;
  // persistent kernel: workgroups that walk one tile fewer than the others (the last round of tiles is partial) start up to `stagger`
  // clock ticks late, spread evenly, so that the CUs stop draining their C tiles in lock-step (0 = off)
  int stagger = 0;
  // patch-embedding mode of the persistent kernel (A_MODE = 1): A is a bf16 IMAGE [B,3,hw,hw]; the row m = b*g2 + gy*g + gx of the im2col
  // matrix and its K index (c*p + py)*p + px are resolved by the LDS-DMA source addresses (16-byte pieces = 8 pixels of one image row),
  // the output row is b*(g2+1) + 1 + (m - b*g2) (row 0 of every image is the CLS token, written elsewhere) and R = positional embedding
  // rows 1..g2 (row index (m mod g2) + 1), models/clip/image_encoder.py:91-106
  int i2c_g2 = 0, i2c_g = 0, i2c_p = 0, i2c_hw = 0;
  int i2c_lcr = 0;   // log2(16-byte chunks per patch row) = log2(p / 8)
  int i2c_ltpc = 0;  // log2(K-tiles per channel) = log2(p*p / 64)
  int i2c_rpk = 0;   // image rows per K-tile = 64 / p
  int gm = 0;        // persistent kernel: tile-order group at run time (0 = the kernel's template value); pick_gm()
  int cn = 0;        // persistent kernel: column tiles per column CHUNK (0 = all of them): chunks are the OUTERMOST level of the tile order; pick_cn()
  // BDIR kernels: W in MFMA-fragment order (mmamd_pack_w_frag): block (nb = n / 32, ks = k / 16) = 64 lanes x 16 B, lane (l31, half) holds
  // W[32 nb + l31][16 ks + 8 half .. + 7] -- the first operand of v_mfma_f32_32x32x16_bf16 as one coalesced 1 KiB buffer load, no LDS
  const bf16* Wp = nullptr;
  // TN split-K kernel with CS (weight gradient + bias gradient in one pass): column sums of A (= dY) over this split's contraction rows,
  // written by the column-tile-0 workgroups to cs_out[split * M + m] (NULL = none)
  float* cs_out = nullptr;
};

// x * sigmoid(1.702 x) with the hardware exp2 / rcp (1 ulp each; the result is rounded to bf16 anyway).  A plain
// `/` compiles to the ~10-instruction IEEE division sequence: measured at 29 % of the MLP-up GEMM's time.
__device__ __forceinline__ float quick_gelu(float v) {
  return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.702f * 1.4426950408889634f * v));
}

// Two values at a time: the epilogues run these on 128 accumulator values per lane while the matrix pipe idles -- 27 % of a tile's time for the
// erf form (FLAVA / CoCa MLP-up), 12 % for QuickGELU (CLIP).  The build has no packed fp32 instructions (multimodal_amd/build.py), so a pair takes
// two issue slots; with them the FLAVA step was 0.75 % shorter (24.90 against 25.09 ms), the CLIP forward the same (13.30 against 13.31 ms).
typedef __attribute__((ext_vector_type(2))) float f32x2;
__device__ __forceinline__ f32x2 quick_gelu2(f32x2 v) {  // bit-identical to quick_gelu() per element (same operations in the same order)
  const f32x2 z = v * (-1.702f * 1.4426950408889634f);
  const f32x2 d = f32x2{__builtin_amdgcn_exp2f(z[0]), __builtin_amdgcn_exp2f(z[1])} + 1.0f;
  return v * f32x2{__builtin_amdgcn_rcpf(d[0]), __builtin_amdgcn_rcpf(d[1])};
}
// erf-GELU as 0.5 v + |v| (0.5 - tau(|v|)) [= max(v, 0) - |v| tau], tau = 0.5 (1 - erf(|v| / sqrt 2)) by the Abramowitz-Stegun 7.1.26 rational form (0.5 folded into the
// polynomial, 1 / sqrt 2 into the rcp's argument): no compare / select, 9 issue slots per value where the r01-r05 form (x = |v| / sqrt 2, h = 0.5 v (1 - erf x),
// v >= 0 ? v - h : h) took ~16.  Both are < 1e-7 |v| from the exact GELU; the result is rounded to bf16.
__device__ __forceinline__ f32x2 gelu_erf2(f32x2 v) {
  const f32x2 ax = __builtin_elementwise_abs(v);
  const f32x2 den = __builtin_elementwise_fma(ax, f32x2{0.3275911f * 0.70710678118654752f, 0.3275911f * 0.70710678118654752f}, f32x2{1.0f, 1.0f});
  const f32x2 t = {__builtin_amdgcn_rcpf(den[0]), __builtin_amdgcn_rcpf(den[1])};
  f32x2 poly = __builtin_elementwise_fma(f32x2{0.5f * 1.061405429f, 0.5f * 1.061405429f}, t, f32x2{0.5f * -1.453152027f, 0.5f * -1.453152027f});
  poly = __builtin_elementwise_fma(poly, t, f32x2{0.5f * 1.421413741f, 0.5f * 1.421413741f});
  poly = __builtin_elementwise_fma(poly, t, f32x2{0.5f * -0.284496736f, 0.5f * -0.284496736f});
  poly = __builtin_elementwise_fma(poly, t, f32x2{0.5f * 0.254829592f, 0.5f * 0.254829592f});
  const f32x2 z = (v * (-0.5f * 1.4426950408889634f)) * v;  // -x^2 log2(e), x = v / sqrt 2
  const f32x2 q = (poly * t) * f32x2{__builtin_amdgcn_exp2f(z[0]), __builtin_amdgcn_exp2f(z[1])};  // tau = 0.5 (1 - erf|x|)
  // max(v, 0) - |v| tau = 0.5 v + |v| (0.5 - tau)   (max as an fp32 instruction canonicalises its operand first: two issue slots per value)
  return __builtin_elementwise_fma(ax, f32x2{0.5f, 0.5f} - q, v * 0.5f);
}

// nn.GELU() = 0.5 v (1 + erf(v / sqrt 2)), one value: the SAME operation sequence as gelu_erf2 (every GEMM kernel of the library must round the
// activation identically -- a batch of 8 takes the plain tiled kernel, a batch of 128 the persistent one, and their rows are compared bit for bit).
// libm's erff is ~60 instructions with branches; this is the Abramowitz-Stegun 7.1.26 rational form on the hardware rcp / exp2: |erf error| <= 1.5e-7,
// far below the bf16 rounding of the value that is stored.  Branch-free.
__device__ __forceinline__ float gelu_erf(float v) { return gelu_erf2(f32x2{v, v})[0]; }

// d/du [u sigmoid(1.702 u)] and d/du [u Phi(u)]: the factor the MLP's backward multiplies the incoming gradient with -- two values at a time (r06: packed
// multiplies / adds / fmas like the forward activations above; the per-value form below is the same operation sequence)
__device__ __forceinline__ f32x2 act_grad2_quick(f32x2 u) {
  const f32x2 z = u * (-1.702f * 1.4426950408889634f);
  const f32x2 d = f32x2{__builtin_amdgcn_exp2f(z[0]), __builtin_amdgcn_exp2f(z[1])} + 1.0f;
  const f32x2 sg = {__builtin_amdgcn_rcpf(d[0]), __builtin_amdgcn_rcpf(d[1])};
  const f32x2 w = (u * 1.702f) * (f32x2{1.0f, 1.0f} - sg);
  return __builtin_elementwise_fma(sg, w, sg);  // sg (1 + 1.702 u (1 - sg))
}
__device__ __forceinline__ f32x2 act_grad2_erf(f32x2 u) {
  const f32x2 ax = __builtin_elementwise_abs(u);
  const f32x2 den = __builtin_elementwise_fma(ax, f32x2{0.3275911f * 0.70710678118654752f, 0.3275911f * 0.70710678118654752f}, f32x2{1.0f, 1.0f});
  const f32x2 t = {__builtin_amdgcn_rcpf(den[0]), __builtin_amdgcn_rcpf(den[1])};
  f32x2 poly = __builtin_elementwise_fma(f32x2{0.5f * 1.061405429f, 0.5f * 1.061405429f}, t, f32x2{0.5f * -1.453152027f, 0.5f * -1.453152027f});
  poly = __builtin_elementwise_fma(poly, t, f32x2{0.5f * 1.421413741f, 0.5f * 1.421413741f});
  poly = __builtin_elementwise_fma(poly, t, f32x2{0.5f * -0.284496736f, 0.5f * -0.284496736f});
  poly = __builtin_elementwise_fma(poly, t, f32x2{0.5f * 0.254829592f, 0.5f * 0.254829592f});
  const f32x2 z = (u * (-0.5f * 1.4426950408889634f)) * u;
  const f32x2 ex = {__builtin_amdgcn_exp2f(z[0]), __builtin_amdgcn_exp2f(z[1])};  // exp(-u^2 / 2)
  const f32x2 h = f32x2{0.5f, 0.5f} - (poly * t) * ex;                           // 0.5 - tail = 0.5 erf(|u| / sqrt 2)
  const f32x2 cdf = f32x2{0.5f, 0.5f} + f32x2{__builtin_copysignf(h[0], u[0]), __builtin_copysignf(h[1], u[1])};  // Phi(u), no compare / select
  return __builtin_elementwise_fma(u * 0.3989422804014327f, ex, cdf);            // Phi(u) + u phi(u)
}
__device__ __forceinline__ float act_grad(float u, int mode) { return mode == 1 ? act_grad2_quick(f32x2{u, u})[0] : act_grad2_erf(f32x2{u, u})[0]; }
__device__ __forceinline__ float combine_res(float v, float r, int mode) { return mode == 0 ? v + r : v * act_grad(r, mode); }
// 8 bf16 results x their 8 bf16 residual values (mode 0: +; 1 / 2: x QuickGELU' / GELU' of the saved pre-activation), the mode switch hoisted (wave-uniform)
__device__ __forceinline__ bf16x8 combine_res8(bf16x8 a8, bf16x8 r8, int mode) {
  if (mode == 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) a8[j] = (bf16)((float)a8[j] + (float)r8[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const f32x2 r = {(float)r8[j], (float)r8[j + 1]};
      const f32x2 o = f32x2{(float)a8[j], (float)a8[j + 1]} * (mode == 1 ? act_grad2_quick(r) : act_grad2_erf(r));
      a8[j] = (bf16)o[0]; a8[j + 1] = (bf16)o[1];
    }
  }
  return a8;
}

__device__ __forceinline__ float apply_act(float v, int act) {
  if (act == MMAMD_ACT_QUICKGELU) return quick_gelu(v);
  if (act == MMAMD_ACT_GELU_ERF) return gelu_erf(v);
  return v;
}

// second output of the dual-store GEMM: the activation of the 8 bf16 values just stored to C (row m, columns n..n+7)
__device__ __forceinline__ void store_act_copy(const GemmArgs& p, uint4 v, int m, int n) {
  if (p.C2 == nullptr) return;  // wave-uniform
  bf16x8 a8 = __builtin_bit_cast(bf16x8, v);
  if (p.act2 != MMAMD_ACT_NONE) {  // (wave-uniform; pairs: packed issue, the same values as apply_act per element)
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const f32x2 in = {(float)a8[j], (float)a8[j + 1]};
      const f32x2 o = p.act2 == MMAMD_ACT_QUICKGELU ? quick_gelu2(in) : gelu_erf2(in);
      a8[j] = (bf16)o[0]; a8[j + 1] = (bf16)o[1];
    }
  }
  *reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(p.C2) + (size_t)m * p.ldc2 + n) = __builtin_bit_cast(uint4, a8);
}

// bias add of the epilogues (depends on the column only).  bias_lds (persistent kernel): the tile's 256 bias values, DMA'd into LDS during the K
// loop (the eight 16-byte global loads per lane at the head of the epilogue were an exposed L2 round trip per tile)
template <int MI, int NI, int TM, int TN>
__device__ __forceinline__ void add_bias(f32x16 (&acc)[NI][MI], const GemmArgs& p, int n0, int wn, int lane, const char* bias_lds = nullptr) {
  const int half = lane >> 5;
  // the branch holds the loads only: with the additions inside it the accumulators met their unchanged selves at its end, through copies that spilled
#pragma unroll
  for (int ni = 0; ni < NI; ++ni) {
    f32x4 bv[4] = {};
    if (p.bias != nullptr) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int n = n0 + wn * TN + ni * 32 + 4 * half + 8 * g;
        if (bias_lds != nullptr) bv[g] = *reinterpret_cast<const f32x4*>(bias_lds + (wn * TN + ni * 32 + 4 * half + 8 * g) * 4);  // block-uniform
        else if (n + 3 < p.N) bv[g] = load4(p.bias + n);
      }
    }
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[ni][mi][4 * g + j] += bv[g][j];
  }
}

static int g_gemm_variant = 0;
// per cent of a tile time; measured (tools/gemm_variant_bench.py --staggers 0,30,60,90,120, profiles/r02_gemm_stagger.txt): 60 is the best or
// within 1 % of it on every shape whose last round of tiles is partial (ViT MLP-up -3.6 %, out-proj -8 %, text MLP-up -10.6 %, patch -7.6 %)
static int g_gemm_stagger = 60;
// experiment knobs (mmamd_debug_set_gemm_knob): [0] tile-order group of the grouped kernel (0 = by CU budget, 4, 8); [1] slack-aware stagger, per cent; [2] walk order of the grouped kernel's two problems
static int g_gemm_knob[8] = {0, 0, 0, 0, 0, 0, 0, 0};
void set_rowln_ablation(int code);  // gemm_rowln.hip

// tile-order group (GemmGroupArgs::gm / GemmArgs::gm): the workgroups an XCD runs concurrently walk gm row panels x all column tiles.  Measured
// on MI355X (r04, profiles/r04_tile_order_ab.txt): gm = 2 is the best or within 0.5 % of it on all four projection pairs of the headline step
// (step 13.39 ms with the r03 value 8, 13.30 with row-major order for N <= 1024 only, 13.25 with 2 everywhere): with few row panels per group
// the column tiles of a panel run at the same time, in lock-step, and every K-slice of the panel is fetched into the XCD's L2 once -- MLP-down
// (3 column tiles, a 1.5 MiB panel per 256 rows that no cache level keeps between rounds) 311 -> 301 us, the vision out-projection alone 93.6 -> 86.5 us.
// Tile order of the persistent kernels, one function for the device code and for the host-side check (mmamd_debug_tile_order; tests/test_host_logic.py
// enumerates it over many grids and asserts a bijection): linear id -> (row tile tm, column tile tn) with the column CHUNK (cn column tiles, the last chunk
// possibly narrower) as the outermost level, then groups of gm row tiles, then the chunk's column tiles, row tile innermost.
__host__ __device__ __forceinline__ void tile_order_map(int id, int tiles_m, int tiles_n, int gm, int cn, int& tm, int& tn) {
  const int full = tiles_m * cn;  // tiles of a full-width chunk
  const int nck = (tiles_n + cn - 1) / cn;
  int ck = id / full;
  ck = ck < nck ? ck : nck - 1;
  const int cw = (tiles_n - ck * cn) < cn ? (tiles_n - ck * cn) : cn;  // this chunk's width
  const int idl = id - ck * full;
  const int per_group = gm * cw;
  const int grp = idl / per_group, within = idl - grp * per_group;
  const int gm0 = grp * gm;
  const int rows = (tiles_m - gm0) < gm ? (tiles_m - gm0) : gm;
  const int tnl = within / rows;
  tn = ck * cn + tnl;
  tm = gm0 + (within - tnl * rows);
}

// Column chunking of the tile order (r06).  The W operand of a wide GEMM does not fit an XCD's 4 MiB L2 (MLP-up: 3072 x 768 bf16 = 4.7 MB), so with all
// column tiles in one group every `gm` row panels re-stream the whole of W through the L2 (MLP-up: 463 MB of W fetches against 104 MB of algorithmic
// reads -- the 1.84 x over-fetch of profiles/r04_pmc_mlp_up_kernel.json).  With the column tiles cut into chunks whose W slice (cn x 256 x K bf16) fits
// beside the A panels in flight, and the chunk as the OUTERMOST level of the tile list, an XCD's contiguous slice of the list lies inside one chunk (or
// two, one after the other): its W slice stays resident for the whole launch and the A panels are read once per chunk.  Bytes are energy, and the step is
// energy-limited.  Tile arithmetic does not depend on the order: bit-identical.
static int pick_cn(int tiles_n, int K) {
  if (g_gemm_knob[4] != 0) return g_gemm_knob[4] < 0 ? tiles_n : g_gemm_knob[4];  // mmamd_debug_set_gemm_knob(4, cn): A/B (-1 = no chunking)
  const long long w_bytes = (long long)tiles_n * 256 * K * 2;
  // W fits: one chunk.  Few column tiles (MLP-down: 3 tiles of a 1.5 MB W slice each, K = 3072): no chunking either -- there the concurrent column tiles
  // of a row panel walk K in lock-step and SHARE the A panel's K-slices; cutting them apart re-reads the 310 MB A operand once per chunk (measured
  // r06: the step +0.33 ms with one-tile chunks on that launch)
  if (w_bytes <= 3ll << 20 || tiles_n <= 6) return tiles_n;
  const long long per_tile = 256ll * K * 2;
  int cn = (int)((5ll << 19) / per_tile);                // chunks of <= 2.5 MiB of W
  if (cn < 1) cn = 1;
  const int nchunk = (tiles_n + cn - 1) / cn;
  return (tiles_n + nchunk - 1) / nchunk;                // equal-width chunks (the last one may be one tile narrower)
}
static int pick_gm(int tiles_n, int cus) {
  if (g_gemm_knob[0] != 0) return g_gemm_knob[0];
  (void)cus;
  return tiles_n <= 4 ? 1 : 2;
}

static unsigned long long* g_gemm_trace = nullptr;
static const void* g_gemm_wp = nullptr;  // experiment (mmamd_debug_set_gemm_wp): fragment-order copy of the NEXT gemm call's W (variants 84 / 85)

// Epilogue shared by the tiled kernels.  Lane owns row m = .. + (lane&31); accumulator regs 4g..4g+3 are columns
// n = .. + 8g + 4*(lane>>5) + {0..3}.
template <int MI, int NI, int TM, int TN, bool OUT_F32, int ACT>
__device__ __forceinline__ void gemm_epilogue(f32x16 (&acc)[NI][MI], const GemmArgs& p, int m0, int n0, int wm, int wn,
                                              int lane) {
  const int l31 = lane & 31, half = lane >> 5;
  // pass 1: bias (depends on n only) or the folded LayerNorm.  pass 2: activation behind ONE uniform branch.  pass 3: residual + store.
  add_bias<MI, NI, TM, TN>(acc, p, n0, wn, lane);
  if constexpr (ACT == MMAMD_ACT_QUICKGELU) {
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float v = acc[ni][mi][r];
          acc[ni][mi][r] = quick_gelu(v);
        }
  } else if constexpr (ACT == MMAMD_ACT_GELU_ERF) {
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float v = acc[ni][mi][r];
          acc[ni][mi][r] = gelu_erf(v);
        }
  }
  const bool has_res = p.R != nullptr;
#pragma unroll
  for (int mi = 0; mi < MI; ++mi) {
    const int m = m0 + wm * TM + mi * 32 + l31;
    const bool mok = m < p.M;
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
      const int nb = n0 + wn * TN + ni * 32 + 4 * half;
      f32x4 v[4];
      // the four residual vectors of this 32 x 32 block: unconditional loads on clamped addresses, all issued before the first is used (r06: loaded
      // inside the lane's bounds branch and used at once, each of them was an exposed round trip -- `s_waitcnt vmcnt(0)` behind every load)
      f32x4 rv4[4];
      if (has_res) {
        const int mc = mok ? m : p.M - 1;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int nc = (nb + 8 * g + 3 < p.N) ? nb + 8 * g : 0;
          if constexpr (OUT_F32) rv4[g] = load4(reinterpret_cast<const float*>(p.R) + (size_t)mc * p.ldr + nc);
          else rv4[g] = load4(reinterpret_cast<const bf16*>(p.R) + (size_t)mc * p.ldr + nc);
        }
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int n = nb + 8 * g;
        const bool ok = mok && (n + 3 < p.N);
        f32x4 t;
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = acc[ni][mi][4 * g + j];
        if (has_res) {
          const f32x4 rv = rv4[g];
#pragma unroll
          for (int j = 0; j < 4; ++j) t[j] = OUT_F32 ? t[j] + rv[j] : combine_res(t[j], rv[j], p.res_mode);
        }
        if constexpr (OUT_F32) {
          if (ok) store4(reinterpret_cast<float*>(p.C) + (size_t)m * p.ldc + n, t);
        }
        v[g] = t;
      }
      if constexpr (!OUT_F32) {
        // pack to bf16 and widen the stores: groups (g, g+1) -> one 16-byte store per lane (T21)
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
          bf16x4 pa, pb;
#pragma unroll
          for (int j = 0; j < 4; ++j) { pa[j] = (bf16)v[g][j]; pb[j] = (bf16)v[g + 1][j]; }
          uint2 ua = __builtin_bit_cast(uint2, pa), ub = __builtin_bit_cast(uint2, pb);
          // lanes 32-63 of `ua` <-> lanes 0-31 of `ub`
          auto s0 = __builtin_amdgcn_permlane32_swap(ua.x, ub.x, false, false);
          auto s1 = __builtin_amdgcn_permlane32_swap(ua.y, ub.y, false, false);
          const uint4 o = make_uint4(s0[0], s1[0], s0[1], s1[1]);
          // lower half now holds columns 8g..8g+7 of its row, upper half columns 8(g+1)..8(g+1)+7
          const int n = n0 + wn * TN + ni * 32 + 8 * (g + half);
          if (mok && n + 7 < p.N) {
            *reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(p.C) + (size_t)m * p.ldc + n) = o;
            store_act_copy(p, o, m, n);
          }
        }
      }
    }
  }
}

// LDS-staged epilogue (used by the pipelined kernels).  The MFMA layout gives every lane 4 consecutive columns of
// ONE row, so a direct store instruction touches 32 different rows with 32 bytes each — measured (ablation: no epilogue)
// at 30-50 % of the kernel time.  Here every wave transposes its sub-tile through a private LDS strip, 32 rows at a
// time, and then stores/loads FULL rows: one wave-instruction covers 8 rows x 128 B (bf16) or 4 rows x 256 B (fp32),
// i.e. whole cache lines; the fp32 residual is read with the same row-contiguous pattern.
template <int MI, int NI, int TM, int TN, bool OUT_F32, int ACT, int ABL = 0>
__device__ __forceinline__ void gemm_epilogue_lds(f32x16 (&acc)[NI][MI], const GemmArgs& p, int m0, int n0, int wm,
                                                  int wn, int lane, int wave, char* smem) {
  static_assert(TN == 64, "row strip below is laid out for 64-column wave tiles");
  const int l31 = lane & 31, half = lane >> 5;
  add_bias<MI, NI, TM, TN>(acc, p, n0, wn, lane);
  if constexpr (ACT == MMAMD_ACT_QUICKGELU) {
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {  // (bit-identical to quick_gelu() per value)
          const f32x2 qg = quick_gelu2(f32x2{acc[ni][mi][r], acc[ni][mi][r + 1]});
          acc[ni][mi][r] = qg[0]; acc[ni][mi][r + 1] = qg[1];
        }
  }
  // erf-GELU is applied where the values are packed for the strip (32x32 at a time): as one pass over all 256
  // accumulators its temporaries spilled (282 VGPRs)
  constexpr int ROWB = OUT_F32 ? (TN * 4 + 16) : (TN * 2 + 16);  // padded strip row: 272 B / 144 B (conflict-free b128)
  const int nw0 = n0 + wn * TN;
  const bool has_res = OUT_F32 && p.R != nullptr;
  f32x4 rr[8], rn[8];
  auto res_load = [&](int mi, f32x4 (&dst)[8]) {
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      // unconditional, on a clamped address (a lane past the edge reads a value it never uses): the predicated form merged the loaded registers with a
      // zero initialisation at the branch join, i.e. `s_waitcnt vmcnt(0)` right behind the loads -- the slab-ahead prefetch below did not exist (r06)
      int m = m0 + wm * TM + mi * 32 + it * 4 + (lane >> 4), n = nw0 + (lane & 15) * 4;
      m = m < p.M ? m : p.M - 1;
      n = n + 3 < p.N ? n : 0;
      dst[it] = load4(reinterpret_cast<const float*>(p.R) + (size_t)m * p.ldr + n);
    }
  };
  if constexpr (OUT_F32) {
    if (has_res) res_load(0, rr);  // in flight across the barrier and the first transpose
  }
  // bf16 output with a bf16 epilogue operand R (+= R, or x act'(R): the MLP's backward): the 32-row slab's four 16-byte loads per lane are issued
  // one slab ahead, UNCONDITIONALLY on clamped addresses (r06: loaded inside the lane's bounds branch and used at once they were sixteen exposed
  // round trips per tile, `s_waitcnt vmcnt(0)` behind each -- see the persistent kernel's descriptor form)
  [[maybe_unused]] uint4 rb[2][4];
  [[maybe_unused]] auto rb_load = [&](int mi, int w) __attribute__((always_inline)) {
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      int m = m0 + wm * TM + mi * 32 + it * 8 + (lane >> 3), n = nw0 + (lane & 7) * 8;
      m = m < p.M ? m : p.M - 1;
      n = n + 7 < p.N ? n : 0;
      rb[w][it] = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(p.R) + (size_t)m * p.ldr + n);
    }
  };
  constexpr bool RB = !OUT_F32 && TN == 64;
  const bool has_rb = RB && p.R != nullptr;
  if constexpr (RB) {
    if (has_rb) rb_load(0, 0);
  }
  __syncthreads();  // every wave is done reading the operand stages: LDS can be reused
  char* strip = smem + wave * (32 * ROWB);
#pragma unroll
  for (int mi = 0; mi < MI; ++mi) {
    const int mrow0 = m0 + wm * TM + mi * 32;
    if constexpr (OUT_F32) {
#pragma unroll
      for (int ni = 0; ni < NI; ++ni)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f32x4 t;
#pragma unroll
          for (int j = 0; j < 4; ++j) t[j] = ACT == MMAMD_ACT_GELU_ERF ? gelu_erf(acc[ni][mi][4 * g + j]) : acc[ni][mi][4 * g + j];
          *reinterpret_cast<f32x4*>(strip + l31 * ROWB + (ni * 32 + 8 * g + 4 * half) * 4) = t;
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      f32x4 vv[8];
#pragma unroll
      for (int it = 0; it < 8; ++it)  // 4 rows x 256 B per wave-instruction
        vv[it] = *reinterpret_cast<const f32x4*>(strip + (it * 4 + (lane >> 4)) * ROWB + (lane & 15) * 16);
      // residual of the NEXT 32-row slab is requested before this slab is consumed: the (otherwise fully exposed)
      // HBM/L2 round trip of every slab overlaps the previous slab's adds and stores (r01 trace: 39k of 72k ticks)
      if (has_res && mi + 1 < MI) res_load(mi + 1, rn);
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const int m = mrow0 + it * 4 + (lane >> 4), n = nw0 + (lane & 15) * 4;
        const bool ok = m < p.M && n + 3 < p.N && ((ABL & 16) == 0 || vv[it][0] == 1.2345678e33f);
        f32x4 v = vv[it];
        if (ok) {
          if (has_res) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += rr[it][j];
          }
          store4(reinterpret_cast<float*>(p.C) + (size_t)m * p.ldc + n, v);
        }
      }
#pragma unroll
      for (int it = 0; it < 8; ++it) rr[it] = rn[it];
    } else {
#pragma unroll
      for (int ni = 0; ni < NI; ++ni)
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
          bf16x4 pa, pb;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float va = acc[ni][mi][4 * g + j], vb = acc[ni][mi][4 * (g + 1) + j];
            if constexpr (ACT == MMAMD_ACT_GELU_ERF) { const f32x2 ge = gelu_erf2(f32x2{va, vb}); va = ge[0]; vb = ge[1]; }
            pa[j] = (bf16)va; pb[j] = (bf16)vb;
          }
          uint2 ua = __builtin_bit_cast(uint2, pa), ub = __builtin_bit_cast(uint2, pb);
          auto s0 = __builtin_amdgcn_permlane32_swap(ua.x, ub.x, false, false);
          auto s1 = __builtin_amdgcn_permlane32_swap(ua.y, ub.y, false, false);
          // lower half: columns 8g..8g+7 of its row; upper half: columns 8(g+1)..8(g+1)+7
          *reinterpret_cast<uint4*>(strip + l31 * ROWB + (ni * 32 + 8 * (g + half)) * 2) = make_uint4(s0[0], s1[0], s0[1], s1[1]);
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if constexpr (RB) {
        if (has_rb && mi + 1 < MI) rb_load(mi + 1, (mi + 1) & 1);
      }
#pragma unroll
      for (int it = 0; it < 4; ++it) {  // 8 rows x 128 B per wave-instruction
        const int row = it * 8 + (lane >> 3), c = lane & 7;
        uint4 v = *reinterpret_cast<const uint4*>(strip + row * ROWB + c * 16);
        const int m = mrow0 + row, n = nw0 + c * 8;
        if constexpr (RB) {
          if (has_rb) v = __builtin_bit_cast(uint4, combine_res8(__builtin_bit_cast(bf16x8, v), __builtin_bit_cast(bf16x8, rb[mi & 1][it]), p.res_mode));
        }
        if (m < p.M && n + 7 < p.N && ((ABL & 16) == 0 || v.x == 0x12345678u)) {
          if (!RB && p.R != nullptr) {
            const uint4 rr = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(p.R) + (size_t)m * p.ldr + n);
            bf16x8 a8 = __builtin_bit_cast(bf16x8, v), r8 = __builtin_bit_cast(bf16x8, rr);
            a8 = combine_res8(a8, r8, p.res_mode);
            v = __builtin_bit_cast(uint4, a8);
          }
          *reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(p.C) + (size_t)m * p.ldc + n) = v;
          store_act_copy(p, v, m, n);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // strip reads done before the next 32 rows overwrite it
  }
}

// LDS-DMA piece through inline asm: 1 KiB (64 lanes x 16 B) from per-lane global addresses to the wave-uniform LDS
// byte address `lds_dst`.  hipcc does not model it (no LDS-alias drain of lgkmcnt before it, no vmcnt bookkeeping):
// completion is counted by hand with s_waitcnt vmcnt(N).  M0 is saved/restored inside the statement (guide 5.7).
__device__ __forceinline__ void dma_piece(const void* gsrc, uint32_t lds_dst) {
  uint32_t keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "v"(gsrc), "s"(lds_dst)
               : "memory");
}

// Same piece with the address split as SCALAR base (SGPR pair) + per-lane 32-bit byte offset: no VALU per piece.
__device__ __forceinline__ void dma_piece_s(const void* sbase, uint32_t voff, uint32_t lds_dst) {
  // M0 is written and consumed inside the statement and NOT restored: nothing else in these kernels uses M0 (no LDS-DMA
  // builtin, no s_movrel, no GWS), so the guide's save/restore pair (2 of 5 scalar instructions per piece) is dropped.
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(voff), "s"(sbase), "s"(lds_dst) : "memory");
}

// 16-byte global store with an explicit cache policy.  POLICY 0: plain (line stays in the XCD's L2); 1: sc1 (written
// through and dropped from L2 - the C tile is never re-read by this kernel, so it should not evict operand panels);
// 2: nt.  The trailing s_nop covers the data-register hazard of an asm store (guide 5.7).
template <int POLICY>
__device__ __forceinline__ void store16(void* ptr, uint4 v) {
  typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;
  const u32x4_t w = __builtin_bit_cast(u32x4_t, v);
  if constexpr (POLICY == 1) asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" : : "v"(ptr), "v"(w) : "memory");
  else if constexpr (POLICY == 2) asm volatile("global_store_dwordx4 %0, %1, off nt\n\ts_nop 1" : : "v"(ptr), "v"(w) : "memory");
  else *reinterpret_cast<uint4*>(ptr) = v;
}

// BM x BN block tile, WM x WN waves, BK = 64
template <int BM, int BN, int WM, int WN, bool OUT_F32, int ACT, bool SGB>
__global__ __launch_bounds__(WM* WN * 64) void gemm_bf16_nt_kernel(const GemmArgs p) {
  constexpr int NW = WM * WN;
  constexpr int TM = BM / WM, TN = BN / WN;
  constexpr int MI = TM / 32, NI = TN / 32;
  constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES;
  constexpr int A_INSTR = BM / 8 / NW, B_INSTR = BN / 8 / NW;  // 1-KiB DMA pieces per wave per stage
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "tile rows must split evenly over the waves");
  static_assert(NW % 4 == 0, "swizzle phase below assumes the wave count is a multiple of 4");
  extern __shared__ __attribute__((aligned(16))) char smem[];

  // ---- block -> tile, XCD-aware (block b runs on XCD b % 8: give each XCD a contiguous id range)
  int bid = blockIdx.x;
  {
    const int nwg = gridDim.x, q = nwg >> 3, r = nwg & 7, xcd = bid & 7, loc = bid >> 3;
    bid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + loc;
  }
  const int tm = bid / p.tiles_n, tn = bid - tm * p.tiles_n;
  const int m0 = tm * BM, n0 = tn * BN;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave - wm * WN;

  // ---- DMA source offsets (bytes from A / W) for this lane; piece i = wave + NW*j covers tile rows 8i..8i+7
  // LDS position of lane: bank row Rr = 4i + (lane>>4), slot' = lane&15; it must hold slot = slot' ^ (Rr&15)
  const int sw = (4 * (wave & 3) + (lane >> 4)) & 15;
  const int slot = (lane & 15) ^ sw;
  const int row8 = 2 * (lane >> 4) + (slot >> 3);  // row inside the 8-row piece
  const int chunk = slot & 7;                      // 16-byte chunk inside the 128-byte row
  uint32_t a_off[A_INSTR], b_off[B_INSTR];
#pragma unroll
  for (int j = 0; j < A_INSTR; ++j) {
    int r = m0 + 8 * (wave + NW * j) + row8;
    r = r < p.M ? r : p.M - 1;
    a_off[j] = ((uint32_t)r * (uint32_t)p.lda + chunk * 8) * 2u;
  }
#pragma unroll
  for (int j = 0; j < B_INSTR; ++j) {
    int r = n0 + 8 * (wave + NW * j) + row8;
    r = r < p.N ? r : p.N - 1;
    b_off[j] = ((uint32_t)r * (uint32_t)p.ldw + chunk * 8) * 2u;
  }
  const char* Ab = reinterpret_cast<const char*>(p.A);
  const char* Wb = reinterpret_cast<const char*>(p.W);

  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u32p)smem;
  auto issue_stage = [&](int buf, int kt) __attribute__((always_inline)) {  // scalar base + K offset, per-lane 32-bit offset: no VALU per piece
    const uint32_t dst = lds0 + buf * STAGE + wave * 1024;
#pragma unroll
    for (int j = 0; j < A_INSTR; ++j) dma_piece_s(Ab + (size_t)kt * 128, a_off[j], dst + NW * j * 1024);
#pragma unroll
    for (int j = 0; j < B_INSTR; ++j) dma_piece_s(Wb + (size_t)kt * 128, b_off[j], dst + A_BYTES + NW * j * 1024);
  };

  // ---- fragment read offsets: lane reads row (lane&31) of a 32-row block, 16-byte chunk 2t + (lane>>5)
  const int l31 = lane & 31, half = lane >> 5;
  const int hsw = l31 >> 1;
  int roff[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) roff[t] = hsw * 256 + (((((l31 & 1) << 3) | (2 * t + half)) ^ hsw) << 4);

  f32x16 acc[NI][MI];
#pragma unroll
  for (int ni = 0; ni < NI; ++ni)
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[ni][mi][r] = 0.f;

  const int KT = p.K >> 6;
  issue_stage(0, 0);
  for (int kt = 0; kt < KT; ++kt) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's DMA pieces of tile kt have landed
    __syncthreads();                                   // ... everyone's; and tile kt-1's reads are done
    if (kt + 1 < KT) issue_stage((kt + 1) & 1, kt + 1);
    const char* sa = smem + (kt & 1) * STAGE + (wm * TM) * 128;
    const char* sb = smem + (kt & 1) * STAGE + A_BYTES + (wn * TN) * 128;
    // register double buffer: fragments of k-step t+1 are in flight while the MFMAs of k-step t issue
    bf16x8 xa[2][MI], wb[2][NI];
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) wb[0][ni] = *reinterpret_cast<const bf16x8*>(sb + ni * 32 * 128 + roff[0]);
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) xa[0][mi] = *reinterpret_cast<const bf16x8*>(sa + mi * 32 * 128 + roff[0]);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int cur = t & 1, nxt = cur ^ 1;
      if (t < 3) {
#pragma unroll
        for (int ni = 0; ni < NI; ++ni)
          wb[nxt][ni] = *reinterpret_cast<const bf16x8*>(sb + ni * 32 * 128 + roff[t + 1]);
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
          xa[nxt][mi] = *reinterpret_cast<const bf16x8*>(sa + mi * 32 * 128 + roff[t + 1]);
      }
#pragma unroll
      for (int ni = 0; ni < NI; ++ni)
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
          acc[ni][mi] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[cur][ni], xa[cur][mi], acc[ni][mi], 0, 0, 0);
    }
    if constexpr (SGB) {
      // pin the software pipeline hipcc otherwise collapses (it re-uses the fragment registers and issues
      // every ds_read AFTER the MFMAs of the step): fragments(t=0); then per k-step one ds_read of step t+1
      // behind each of the first NI+MI MFMAs of step t.   masks: MFMA = 0x008, DS read = 0x100
      constexpr int NF = NI + MI, NM = NI * MI;
      __builtin_amdgcn_sched_group_barrier(0x100, NF, 0);
#pragma unroll
      for (int t = 0; t < 3; ++t) {
#pragma unroll
        for (int i = 0; i < NF; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        if constexpr (NM > NF) __builtin_amdgcn_sched_group_barrier(0x008, NM - NF, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, NM, 0);
    }
  }

  gemm_epilogue<MI, NI, TM, TN, OUT_F32, ACT>(acc, p, m0, n0, wm, wn, lane);
}


// ---------------------------------------------------------------------------------------------------------
// Pipelined kernel ("P"): same tile geometry / LDS image / epilogue as above, different schedule.
//   * the K loop is ROTATED across the barrier: the 4th k-step's MFMAs of tile k are issued AFTER the barrier
//     that publishes tile k+1, so they cover the barrier release, the LDS-DMA issue for tile k+2 and the
//     latency of the first fragment reads of tile k+1 (in the plain loop the matrix pipe idles through all
//     three on every K-tile: SQ_WAIT_ANY was 35 % of wave cycles there);
//   * the 8 DMA pieces of the next tile are interleaved one-per-MFMA instead of issued as a burst;
//   * block -> tile order is grouped (GM row-panels x all column tiles per group) inside each XCD's contiguous
//     id range, so the ~32 blocks an XCD runs concurrently share GM activation panels and ~32/GM weight tiles
//     in its 4 MiB L2 (the row-major order re-fetched the whole weight matrix every 32 blocks: FETCH_SIZE was
//     3-6x the algorithmic bytes).
// ABL (ablation bit mask, perf experiments only — results are WRONG for ABL != 0): 1 = no DMA in the loop,
// 2 = no MFMA, 4 = no epilogue, 8 = no fragment reads, 16 = no global accesses in the epilogue
// TNM ("TN" operands, weight gradients): C[M,N] = sum_t A[t][m] W[t][n] with A = [K, lda] and W = [K, ldw] ROW-major over the
// contraction index t (dW = dY^T X straight from the row-major dY and X: no transposed bf16 copies in HBM).  The LDS image of a
// K-tile is then [64 t][256 cols], stored as 256-byte units of [4 t][32 cols] (two [4][16] blocks) in [t/4][cols/32] order — the
// DMA lays it out through its per-lane source addresses — and every MFMA operand is two ds_read_b64_tr_b16 (4 + 4 contraction
// indices of one column per lane; the two 16-lane groups of a half-wave read one contiguous 256-byte unit: conflict-free).
template <int BM, int BN, int WM, int WN, bool OUT_F32, int ACT, int GM, int ABL = 0, bool LDSEPI = true, bool TNM = false, int SCH = 0, bool CS = false>
__global__ __launch_bounds__(WM* WN * 64) void gemm_bf16_nt_kernel_p(const GemmArgs p, const int tiles_m,
                                                                        unsigned long long* trace = nullptr) {
  int bid = blockIdx.x;
  const int nwg = gridDim.x, bid_launch = blockIdx.x, split_y = blockIdx.y;
#include "gemm_p_body.inc"
}


// Grouped weight gradients (r05): up to 8 TN split-K problems in ONE launch -- the four dW = dY^T X of a transformer layer.  Launched one by one, the
// small ones need 21-28 splits to fill 256 CUs (28 K-tiles per workgroup between a 64 KiB prologue and a 256 KiB partial store; 66 MB of partials per
// GEMM whatever its size) and each pays its own reduce launch; together they fill the chip at a few splits each.  Problem i owns the workgroups
// [wg0[i], wg0[i] + nwg[i]) (wg0 8-aligned, so a workgroup's XCD is its local index mod 8 as in the plain launch); the padding workgroups exit.
constexpr int kTnGroupMax = 8;
struct GemmTnGroupArgs {
  GemmArgs p[kTnGroupMax];
  int wg0[kTnGroupMax], nwg[kTnGroupMax], tiles_m[kTnGroupMax];
  int nprob;
};
template <bool CS>
__global__ __launch_bounds__(512) void gemm_bf16_tn_group_kernel(const GemmTnGroupArgs g) {
  constexpr int BM = 256, BN = 256, WM = 2, WN = 4, ACT = MMAMD_ACT_NONE, GM = 8, ABL = 0, SCH = 0;
  constexpr bool OUT_F32 = true, LDSEPI = true, TNM = true;
  int pi = 0;
#pragma unroll
  for (int i = 1; i < kTnGroupMax; ++i)
    if (i < g.nprob && (int)blockIdx.x >= g.wg0[i]) pi = i;
  pi = __builtin_amdgcn_readfirstlane(pi);
  int bid = (int)blockIdx.x - g.wg0[pi];
  const int nwg = g.nwg[pi];
  if (bid >= nwg) return;
  const GemmArgs& p = g.p[pi];
  const int tiles_m = g.tiles_m[pi], bid_launch = blockIdx.x, split_y = 0;
  unsigned long long* const trace = nullptr;
#include "gemm_p_body.inc"
}



#ifdef MMAMD_EXPERIMENTS
#include "experiments/gemm_kernels_gqs.inc"  // schedule experiments G / Q / S (not faster: DESIGN.md 4.1)
#endif

// ---------------------------------------------------------------------------------------------------------
// Persistent pipelined kernel ("PP", the production kernel): the P schedule, but ONE workgroup per CU walks the tiles
// vb = blockIdx.x, + gridDim.x, ...  The r01 section trace of P showed 6 % of every tile in the exposed first-stage
// load and 22-55 % in the epilogue; here the first K-tile of the NEXT output tile is DMA'd (into ring buffer 0, free
// during the last K-tile) behind the last K-tile's MFMAs, so it lands while the epilogue runs out of ring buffer 1.
//   * epilogue strips live in ring buffer 1 only (32 rows x 128 B per wave and pass, fp32 tiles in two column halves)
//   * the fp32 residual of pass i+1 is requested before pass i is consumed
//   * tile order: same XCD-contiguous, GM-grouped order as P, applied to the virtual block id (gridDim.x % 8 == 0)
// WM x WN waves: 2 x 4 = eight 128x64 wave tiles (two waves per SIMD), or 2 x 2 = four 128x128 wave tiles (ONE wave per
// SIMD, 256 accumulator registers in the unified VGPR/AGPR file): 8 instead of 12 fragment reads per 16 MFMAs.
template <bool OUT_F32, int ACT, int GM, int WM = 2, int WN = 4, int STP = 0, int RDP = 0, int RES_DEPTH = 1, bool BLDS = false, int A_MODE = 0,
          bool BDIR = false>
__global__ __launch_bounds__(WM* WN * 64) void gemm_bf16_nt_kernel_pp(const GemmArgs p, const int tiles_m, const int ntiles) {
  constexpr int BM = 256, BN = 256, NW = WM * WN;
  constexpr int TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;
  constexpr int A_BYTES = BM * 128, STAGE = (BM + BN) * 128;
  // BDIR: the W fragments never pass through LDS -- every wave loads its own (pre-packed, GemmArgs::Wp) fragments of the NEXT K-tile straight
  // into registers while it computes this one: a third fewer LDS reads per MFMA in the 8-wave form, half in the 4-wave form, half the DMA pieces
  constexpr int A_INSTR = BM / 8 / NW, B_INSTR = BDIR ? 0 : BN / 8 / NW, NDMA = A_INSTR + B_INSTR, NF = (BDIR ? 0 : NI) + MI, NM = NI * MI;
  static_assert(!BDIR || A_MODE == 0, "BDIR: plain A operand only");
  static_assert(NM >= NDMA && NM >= NF && NW % 4 == 0, "interleave needs one MFMA per DMA piece / fragment read");
  constexpr int CH = TN / 64;  // 128-byte column chunks of a wave tile row in bf16
  extern __shared__ __attribute__((aligned(16))) char smem[];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave - wm * WN;
  const int l31 = lane & 31, half = lane >> 5;

  const int GMr = p.gm > 0 ? p.gm : GM;  // (row-major, gm = 1, for few column tiles: see pick_gm)
  const int CNr = p.cn > 0 && p.cn < p.tiles_n ? p.cn : p.tiles_n;  // column tiles per chunk (pick_cn); chunk = outermost level of the order
  auto tile_of = [&](int vb, int& tm, int& tn) __attribute__((always_inline)) {
    const int q = ntiles >> 3, r = ntiles & 7, xcd = vb & 7, loc = vb >> 3;
    const int id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + loc;
    tile_order_map(id, tiles_m, p.tiles_n, GMr, CNr, tm, tn);
  };

  // DMA source offsets of this lane (see kernel above for the swizzle): depend on the tile, not on K
  const int sw = (4 * (wave & 3) + (lane >> 4)) & 15;
  const int slot = (lane & 15) ^ sw;
  const int row8 = 2 * (lane >> 4) + (slot >> 3);
  const int chunk = slot & 7;
  constexpr int B_ARR = B_INSTR > 0 ? B_INSTR : 1;
  auto tile_offsets = [&](int tm, int tn, uint32_t (&ao)[A_INSTR], uint32_t (&bo)[B_ARR]) {
#pragma unroll
    for (int j = 0; j < A_INSTR; ++j) {
      int r = tm * BM + 8 * (wave + NW * j) + row8;
      r = r < p.M ? r : p.M - 1;
      if constexpr (A_MODE == 1) {  // patch row r = (b, gy, gx); this lane's 16-byte chunk = 8 pixels of patch row py_l of the K-tile
        const int b = r / p.i2c_g2, t = r - b * p.i2c_g2;
        const int gy = t / p.i2c_g, gx = t - gy * p.i2c_g;
        const int py_l = chunk >> p.i2c_lcr, px0 = (chunk & ((1 << p.i2c_lcr) - 1)) * 8;
        ao[j] = ((uint32_t)((b * 3 * p.i2c_hw + gy * p.i2c_p + py_l) * p.i2c_hw) + (uint32_t)(gx * p.i2c_p + px0)) * 2u;
      } else {
        ao[j] = ((uint32_t)r * (uint32_t)p.lda + chunk * 8) * 2u;
      }
    }
#pragma unroll
    for (int j = 0; j < B_INSTR; ++j) {
      int r = tn * BN + 8 * (wave + NW * j) + row8;
      r = r < p.N ? r : p.N - 1;
      bo[j] = ((uint32_t)r * (uint32_t)p.ldw + chunk * 8) * 2u;
    }
  };
  const char* Ab = reinterpret_cast<const char*>(p.A);
  const char* Wb = reinterpret_cast<const char*>(p.W);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u32p)smem;
  uint32_t a_off[A_INSTR], b_off[B_ARR], a_nxt[A_INSTR], b_nxt[B_ARR];
  // BDIR: per-lane byte offsets of this wave's NI fragment columns in the packed W (block row nb = column / 32, KS blocks of 1 KiB per row)
  const int KS = p.K >> 4;
  uint32_t bd_off[NI], bd_nxt[NI];
  auto bdir_offsets = [&](int tn, uint32_t (&bo)[NI]) {
    const int nbmax = ((p.N + 31) >> 5) - 1;
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
      int nb = tn * (BN / 32) + wn * NI + ni;
      nb = nb < nbmax ? nb : nbmax;  // column blocks past N are never stored
      bo[ni] = ((uint32_t)nb * (uint32_t)KS * 64u + (uint32_t)lane) * 16u;
    }
  };
  const int32x4 wp_srd = make_srd(BDIR ? p.Wp : p.W, 0x7fffffffu);
  bf16x8 wbd[4][NI];  // BDIR: W fragments, one slot per k-step of a K-tile (reloaded as soon as its MFMAs are issued)
  auto issue_piece = [&](int buf, int kt, int i) __attribute__((always_inline)) {
    const uint32_t dst = lds0 + buf * STAGE + (i < A_INSTR ? (wave + NW * i) * 1024 : A_BYTES + (wave + NW * (i - A_INSTR)) * 1024);
    if (i < A_INSTR) {
      if constexpr (A_MODE == 1) {  // K-tile kt = channel kt >> ltpc, image rows (kt & mask) * rpk .. + rpk - 1 of every patch
        const size_t koff = ((size_t)(kt >> p.i2c_ltpc) * p.i2c_hw * p.i2c_hw + (size_t)(kt & ((1 << p.i2c_ltpc) - 1)) * p.i2c_rpk * p.i2c_hw) * 2u;
        dma_piece_s(Ab + koff, a_off[i], dst);
      } else {
        dma_piece_s(Ab + (size_t)kt * 128, a_off[i], dst);
      }
    } else {
      if constexpr (!BDIR) dma_piece_s(Wb + (size_t)kt * 128, b_off[i - A_INSTR], dst);
    }
  };
  // The W loads and every wait on them are inline asm: the compiler's wait insertion does not see the asm DMA pieces and (measured on the ISA)
  // merges the loop paths into vmcnt(3) / vmcnt(0) waits that land behind the DMA issue of the next K-tile.  The waits are tied to the slot
  // registers ("+v"), so no MFMA that reads a slot can move above its wait; nothing but v_mfma may read a slot between its load and its wait
  // (tools/check_bdir_isa.py checks the ISA for that).
  auto bdir_load = [&](auto tc, int ni, uint32_t voff, int kt) __attribute__((always_inline)) {
    constexpr int T = decltype(tc)::value;
    bf16x8& d = wbd[T][ni];  // (asm operands inside a generic lambda must be the lambda's own names)
    const int32x4 srd = wp_srd;
    const int soff = (kt * 4 + T) * 1024;
    asm volatile("buffer_load_dwordx4 %0, %1, %2, %3 offen" : "=v"(d) : "v"(voff), "s"(srd), "s"(soff) : "memory");
  };
  // (a tied wait inside a branch makes the register allocator COPY the slot on the way in -- a read before the data has landed: the tied waits
  //  are unconditional, the stricter wait of the rare path is an untied statement in front of it)
  auto bdir_wait_plain = [&](auto nc) __attribute__((always_inline)) {
    constexpr int N = decltype(nc)::value;
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
  };
  auto bdir_wait = [&](auto tc, auto nc) __attribute__((always_inline)) {  // s_waitcnt vmcnt(N) ahead of the readers of slot T
    constexpr int T = decltype(tc)::value, N = decltype(nc)::value;
    static_assert(NI == 2 || NI == 4, "slot width");
    bf16x8(&w)[NI] = wbd[T];
    if constexpr (NI == 2) asm volatile("s_waitcnt vmcnt(%2)" : "+v"(w[0]), "+v"(w[1]) : "n"(N));
    else asm volatile("s_waitcnt vmcnt(%4)" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]) : "n"(N));
  };
  // output / residual row of GEMM row m (A_MODE = 1: the token row behind its image's CLS row; positional-embedding row of the patch)
  auto c_row = [&](int m) -> size_t { if constexpr (A_MODE == 1) return (size_t)m + (size_t)(m / p.i2c_g2) + 1; else return (size_t)m; };
  auto r_row = [&](int m) -> size_t { if constexpr (A_MODE == 1) return (size_t)(m % p.i2c_g2) + 1; else return (size_t)m; };

  const int hsw = l31 >> 1;
  uint32_t ra[2][4], rb[2][4];
#pragma unroll
  for (int bf = 0; bf < 2; ++bf)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t ro = hsw * 256 + (((((l31 & 1) << 3) | (2 * t + half)) ^ hsw) << 4);
      ra[bf][t] = lds0 + bf * STAGE + (wm * TM) * 128 + ro;
      rb[bf][t] = lds0 + bf * STAGE + A_BYTES + (wn * TN) * 128 + ro;
    }
  typedef __attribute__((address_space(3))) const bf16x8* lds_frag_p;

  f32x16 acc[NI][MI];
  bf16x8 xa0[MI], wb0[NI], xa1[MI], wb1[NI];
  auto load_frags = [&](auto bufc, int t, bf16x8 (&xa)[MI], bf16x8 (&wb)[NI]) {
    constexpr int BF = decltype(bufc)::value;
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) wb[ni] = *reinterpret_cast<lds_frag_p>((uintptr_t)(rb[BF][t] + ni * 32 * 128));
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) xa[mi] = *reinterpret_cast<lds_frag_p>((uintptr_t)(ra[BF][t] + mi * 32 * 128));
  };
  auto mma = [&](bf16x8 (&xa)[MI], bf16x8 (&wb)[NI]) {
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
        acc[ni][mi] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[ni], xa[mi], acc[ni][mi], 0, 0, 0);
  };
  auto mma_one = [&](bf16x8 (&xa)[MI], bf16x8 (&wb)[NI], int i) {
    acc[i / MI][i % MI] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[i / MI], xa[i % MI], acc[i / MI][i % MI], 0, 0, 0);
  };
  // one K-tile out of ring buffer BF; behind the first MFMA group one DMA piece each of (ktsrc -> buffer BF^1)
  auto tile_body = [&](auto bufc, int ktsrc, const bool issue) __attribute__((always_inline)) {
    constexpr int BF = decltype(bufc)::value;
    load_frags(bufc, 0, xa0, wb0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      mma_one(xa1, wb1, i);
      if (issue && i < NDMA) issue_piece(BF ^ 1, ktsrc, i);  // wave-uniform scalar branch
      __builtin_amdgcn_sched_barrier(0);
    }
    load_frags(bufc, 1, xa1, wb1);
    mma(xa0, wb0);
    load_frags(bufc, 2, xa0, wb0);
    mma(xa1, wb1);
    load_frags(bufc, 3, xa1, wb1);
    mma(xa0, wb0);
#pragma unroll
    for (int t = 0; t < 3; ++t) {
      if constexpr (RDP == 0) {         // one read of the next k-step behind each of the first NF MFMAs
#pragma unroll
        for (int i = 0; i < NF; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        if constexpr (NM > NF) __builtin_amdgcn_sched_group_barrier(0x008, NM - NF, 0);
      } else if constexpr (RDP == 1) {  // all NF reads in one burst behind the first MFMA (maximum cover)
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, NF, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, NM - 1, 0);
      } else {                          // two reads behind each of the first NF/2 MFMAs
#pragma unroll
        for (int i = 0; i < NF / 2; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, NM - NF / 2, 0);
      }
    }
  };
  // BDIR form of the K-tile kt (in ring buffer BF): A fragments from LDS as above, W fragments from the register slots wbd[t].  Slot t is reloaded
  // right behind the MFMAs that read it: slot 3 (read by the rotated k-step of K-tile kt - 1 in the first group) <- W(kt, 3), slots 0 .. 2 <- W(ktsrc, t)
  // -- every load has three to four k-steps (>= 1500 cycles) to land.  `last`: ktsrc belongs to the NEXT output tile (offsets bd_nxt).
  auto tile_body_bdir = [&](auto bufc, int kt, int ktsrc, const bool issue, const bool last) __attribute__((always_inline)) {
    constexpr int BF = decltype(bufc)::value;
    using T0 = std::integral_constant<int, 0>;
    using T1 = std::integral_constant<int, 1>;
    using T2 = std::integral_constant<int, 2>;
    using T3 = std::integral_constant<int, 3>;
    // VMEM issue order of a body: DMA x NDMA (if `issue`), slot 3 x NI, slot 0 x NI, slot 1 x NI, slot 2 x NI.  The readers of slot t (loaded one body
    // ago) may leave everything younger in flight: the rest of that body's reloads + this body's issues so far
    using W_ISSUE = std::integral_constant<int, 3 * NI + NDMA>;  // step 0: slots 1, 2 of the last body + DMA + slot 3;  steps 1, 2: the same count
    using W_QUIET = std::integral_constant<int, 3 * NI>;         // ... without DMA pieces in this body (the last K-tile of the last tile)
    auto load_a = [&](int t, bf16x8 (&xa)[MI]) __attribute__((always_inline)) {
#pragma unroll
      for (int mi = 0; mi < MI; ++mi) xa[mi] = *reinterpret_cast<lds_frag_p>((uintptr_t)(ra[BF][t] + mi * 32 * 128));
    };
    load_a(0, xa0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      mma_one(xa1, wbd[3], i);
      if (issue && i < NDMA) issue_piece(BF ^ 1, ktsrc, i);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) bdir_load(T3{}, ni, bd_off[ni], kt);
    uint32_t bn[NI];
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) bn[ni] = last ? bd_nxt[ni] : bd_off[ni];  // (bd_nxt == bd_off when there is no next tile)
    if (!issue) bdir_wait_plain(W_QUIET{});
    bdir_wait(T0{}, W_ISSUE{});
    __builtin_amdgcn_sched_barrier(0);
    load_a(1, xa1);
    mma(xa0, wbd[0]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) bdir_load(T0{}, ni, bn[ni], ktsrc);  // unconditional (see above)
    if (!issue) bdir_wait_plain(W_QUIET{});
    bdir_wait(T1{}, W_ISSUE{});
    __builtin_amdgcn_sched_barrier(0);
    load_a(2, xa0);
    mma(xa1, wbd[1]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) bdir_load(T1{}, ni, bn[ni], ktsrc);
    if (!issue) bdir_wait_plain(W_QUIET{});
    bdir_wait(T2{}, W_ISSUE{});
    __builtin_amdgcn_sched_barrier(0);
    load_a(3, xa1);
    mma(xa0, wbd[2]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) bdir_load(T2{}, ni, bn[ni], ktsrc);
    __builtin_amdgcn_sched_barrier(0);
  };
  using B0 = std::integral_constant<int, 0>;
  using B1 = std::integral_constant<int, 1>;
  // BDIR, `first` = first K-tile of an output tile: the epilogue's stores are in flight too (they do not retire in order with loads): vmcnt(0).
  // Otherwise the DMA pieces of this K-tile and slot 3 must have landed; the reloads of slots 0 .. 2 (3 NI loads, the youngest) may stay in flight.
  // `drain` (r06, see the grouped kernel's sync_first): the number of unconditional buffer loads / stores the previous tile's epilogue issued
  // AFTER the DMA of this tile's first K-tile -- the first barrier of a tile waits for that DMA only, not for the epilogue's stores
  int drain = 0;
  auto sync_tile = [&](const bool first = true) __attribute__((always_inline)) {
    if constexpr (BDIR) {
      if (first) bdir_wait_plain(std::integral_constant<int, 0>{});
      bdir_wait(std::integral_constant<int, 3>{}, std::integral_constant<int, 3 * NI>{});
    } else {
      if (first && drain == 16) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
      else if (first && drain == 32) asm volatile("s_waitcnt vmcnt(32)" ::: "memory");
      else if (first && drain == 63) asm volatile("s_waitcnt vmcnt(63)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __syncthreads();
  };

  const int KT = p.K >> 6;  // even (launcher)
  int vb = blockIdx.x;
  int tm, tn;
  tile_of(vb, tm, tn);
  tile_offsets(tm, tn, a_off, b_off);
#pragma unroll
  for (int i = 0; i < NDMA; ++i) issue_piece(0, 0, i);
  if constexpr (BDIR) {
    bdir_offsets(tn, bd_off);
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
#pragma unroll
      for (int j = 0; j < 8; ++j) wbd[3][ni][j] = (bf16)0.f;  // read (times zero) by the first tile's rotated MFMAs
    }
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) bdir_load(std::integral_constant<int, 0>{}, ni, bd_off[ni], 0);
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) bdir_load(std::integral_constant<int, 1>{}, ni, bd_off[ni], 0);
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) bdir_load(std::integral_constant<int, 2>{}, ni, bd_off[ni], 0);
  }
  if (p.stagger > 0) {
    const int heavy = ntiles % (int)gridDim.x;  // workgroups 0 .. heavy-1 walk one tile more: they start at once
    if (heavy > 0 && (int)blockIdx.x >= heavy) {
      const long long delay = (long long)p.stagger * ((int)blockIdx.x - heavy + 1) / ((int)gridDim.x - heavy);
      const long long t0 = __builtin_readcyclecounter();
      while (__builtin_readcyclecounter() - t0 < delay) __builtin_amdgcn_s_sleep(32);
    }
  } else if (p.stagger < 0) {
    // experiment (mmamd_debug_set_gemm_stagger(1000 + percent)): EVERY workgroup is delayed, the 32 of an XCD spread evenly over
    // [0, |stagger|) -- de-synchronises the chip-wide store bursts at the price of up to |stagger| of makespan
    const long long delay = (long long)(-p.stagger) * ((int)blockIdx.x >> 3) / (((int)gridDim.x + 7) >> 3);
    const long long t0 = __builtin_readcyclecounter();
    while (__builtin_readcyclecounter() - t0 < delay) __builtin_amdgcn_s_sleep(32);
  }

  while (true) {
    const int m0 = tm * BM, n0 = tn * BN;
    const int nvb = vb + gridDim.x;
    const bool more = nvb < ntiles;
    int ntm = 0, ntn = 0;
    if (more) {
      tile_of(nvb, ntm, ntn);
      tile_offsets(ntm, ntn, a_nxt, b_nxt);
      if constexpr (BDIR) bdir_offsets(ntn, bd_nxt);
    } else if constexpr (BDIR) {
#pragma unroll
      for (int ni = 0; ni < NI; ++ni) bd_nxt[ni] = bd_off[ni];
    }
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[ni][mi][r] = 0.f;
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int j = 0; j < 8; ++j) xa1[mi][j] = (bf16)0.f;
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
      for (int j = 0; j < 8; ++j) wb1[ni][j] = (bf16)0.f;

#pragma unroll 1
    for (int kt = 0; kt < KT; kt += 2) {
      sync_tile(kt == 0);
      if constexpr (BLDS) {
        // the tile's 256 bias values (1 KiB = one DMA piece, issued by wave 0) land in LDS behind the ring while the K loop runs;
        // same hazards as the statistics above: issued after the tile's first barrier, waited for by the next sync_tile
        if (kt == 0 && wave == 0 && p.bias != nullptr) {
          const uint32_t limit = (uint32_t)(p.N - n0) * 4u - 16u;
          uint32_t off = lane * 16u;
          off = off < limit ? off : limit;  // columns past N (never stored) re-read the last valid 16 bytes
          dma_piece_s(reinterpret_cast<const char*>(p.bias) + (size_t)n0 * 4u, off, lds0 + 2 * STAGE);
        }
      }
      if constexpr (BDIR) tile_body_bdir(B0{}, kt, kt + 1, true, false);
      else tile_body(B0{}, kt + 1, true);
      const bool last = kt + 2 >= KT;
      if (last && more) {  // this tile's loads are all issued: switch the DMA source to the next tile's first K-tile
#pragma unroll
        for (int j = 0; j < A_INSTR; ++j) a_off[j] = a_nxt[j];
#pragma unroll
        for (int j = 0; j < B_INSTR; ++j) b_off[j] = b_nxt[j];
      }
      sync_tile(false);
      if constexpr (BDIR) tile_body_bdir(B1{}, kt + 1, last ? 0 : kt + 2, !last || more, last);
      else tile_body(B1{}, last ? 0 : kt + 2, !last || more);
    }
    if constexpr (BDIR) {
      bdir_wait(std::integral_constant<int, 3>{}, std::integral_constant<int, 3 * NI>{});
      mma(xa1, wbd[3]);  // flush the rotated last k-step
      // the slot 0 .. 2 reloads of the last body are DEAD after the last tile: the compiler may hand their registers to the epilogue while
      // the (asm, invisible) loads are still in flight -- every W load has landed before the epilogue starts
      if (!more) bdir_wait_plain(std::integral_constant<int, 0>{});
      if (more) {
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) bd_off[ni] = bd_nxt[ni];
      }
    } else {
      mma(xa1, wb1);
    }

    // ---------------- epilogue (LDS strips in ring buffer 1; buffer 0 is receiving the next tile) ----------------
    // fp32 residual: a ring of RD passes of loads in flight, the first RD issued here (before the bias / barrier / first transpose).
    // Measured (tools/gemm_variant_bench.py --variants 60,61,62,63, r02): depth 1 = 2 (out-proj 100.7 / 100.5 us), depth 3 and 4
    // LOSE (115 / 133 us: 21 spilled registers and more loads queued per CU) -- the residual's latency is not what the fp32
    // epilogue waits for; the default stays 1.
    constexpr int RD = OUT_F32 ? RES_DEPTH : 1;
    const int nw0 = n0 + wn * TN;
    const int rrow = lane >> 3, rc = (lane & 7) * 4;  // fp32 read-back: 8 rows x 128 B per wave-instruction
    f32x4 rq[RD][4];
    auto res_load = [&](int pass, f32x4 (&dst)[4]) __attribute__((always_inline)) {  // pass = mi * NI + ni
      const int mi = pass / NI, ni = pass - mi * NI;
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        // (unconditional, clamped: a predicated load is waited for at the branch join -- see gemm_epi_f32.inc; lanes past the edge never use the value)
        int m = m0 + wm * TM + mi * 32 + it * 8 + rrow, n = nw0 + ni * 32 + rc;
        m = m < p.M ? m : p.M - 1;
        n = n + 3 < p.N ? n : 0;
        dst[it] = load4(reinterpret_cast<const float*>(p.R) + r_row(m) * p.ldr + n);
      }
    };
    // the pipelined buffer-descriptor epilogue (gemm_epi_f32.inc, r06) serves the plain fp32 output of the 8-wave form; the patch-embedding
    // mode (rows remapped per image) and the 4-wave form keep the predicated loop below
    constexpr bool PIPE = OUT_F32 && A_MODE == 0 && MI * NI == 8;
#define MMAMD_EPI_PART 1
#include "gemm_epi_f32.inc"
    if constexpr (OUT_F32 && !PIPE) {
      if (p.R != nullptr) {
#pragma unroll
        for (int d = 0; d < RD; ++d) res_load(d, rq[d]);
      }
    }
    add_bias<MI, NI, TM, TN>(acc, p, n0, wn, lane, BLDS ? smem + 2 * STAGE : nullptr);
    if constexpr (ACT == MMAMD_ACT_QUICKGELU || (ACT == MMAMD_ACT_GELU_ERF && !OUT_F32)) {  // (activation + fp32 output: inside the fp32 passes; no model path)
#pragma unroll
      for (int ni = 0; ni < NI; ++ni)
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
          for (int r = 0; r < 16; r += 2) {  // adjacent accumulator registers: the pairs need no moves
            const f32x2 in = {acc[ni][mi][r], acc[ni][mi][r + 1]};
            const f32x2 qg = ACT == MMAMD_ACT_QUICKGELU ? quick_gelu2(in) : gelu_erf2(in);
            acc[ni][mi][r] = qg[0]; acc[ni][mi][r + 1] = qg[1];
          }
    }
    constexpr int ROWB = 144;  // 128-byte strip rows + 16 B pad (conflict-free b128 both ways)
    char* strip = smem + STAGE + wave * (32 * ROWB);
    if constexpr (!PIPE) __syncthreads();  // every wave has finished reading the last K-tile out of ring buffer 1 (PIPE: inside the include)
    if constexpr (PIPE) {
#define MMAMD_EPI_PART 2
#include "gemm_epi_f32.inc"
      drain = has_res ? 63 : 32;
    } else if constexpr (OUT_F32) {
      drain = 0;
      const bool has_res = p.R != nullptr;
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) {
          const int pass = mi * NI + ni;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            f32x4 t;
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = ACT == MMAMD_ACT_GELU_ERF ? gelu_erf(acc[ni][mi][4 * g + j]) : acc[ni][mi][4 * g + j];
            *reinterpret_cast<f32x4*>(strip + l31 * ROWB + (8 * g + 4 * half) * 4) = t;
          }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          f32x4 vv[4];
#pragma unroll
          for (int it = 0; it < 4; ++it) vv[it] = *reinterpret_cast<const f32x4*>(strip + (it * 8 + rrow) * ROWB + rc * 4);
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const int m = m0 + wm * TM + mi * 32 + it * 8 + rrow, n = nw0 + ni * 32 + rc;
            const bool ok = m < p.M && n + 3 < p.N;
            f32x4 v = vv[it];
            if (ok) {
              if (has_res) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += rq[pass % RD][it][j];
              }
              store16<STP>(reinterpret_cast<float*>(p.C) + c_row(m) * p.ldc + n, __builtin_bit_cast(uint4, v));
            }
          }
          if (has_res && pass + RD < MI * NI) res_load(pass + RD, rq[pass % RD]);  // refill the slot this pass just consumed
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    } else if (A_MODE == 0 && CH == 1 && MI * 4 == 16 && p.R == nullptr && p.C2 == nullptr) {
      // bf16 output, no residual, no second output: buffer-descriptor stores (the grouped kernel's form), not drained by the next tile's first barrier
      const int mw = m0 + wm * TM;
      const long long rows_left = (long long)p.M - mw;
      const long long cb = rows_left > 0 ? rows_left * p.ldc * 2 : 0;
      const __amdgpu_buffer_rsrc_t c16_srd = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(p.C) + ((size_t)mw * p.ldc + nw0) * 2, 0,
                                                                               cb > 0x7fffffffLL ? 0x7fffffff : (int)cb, 0x00020000);
      const uint32_t c16_lane = ((uint32_t)((lane >> 3) * p.ldc + (lane & 7) * 8) * 2u) | ((nw0 + (lane & 7) * 8 + 7 < p.N) ? 0u : 0x80000000u);
      typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_s;
#pragma unroll
      for (int mi = 0; mi < MI; ++mi) {
#pragma unroll
        for (int nn = 0; nn < 2; ++nn)
#pragma unroll
          for (int g = 0; g < 4; g += 2) {
            const int ni = nn;
            bf16x4 pa, pb;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float va = acc[ni][mi][4 * g + j], vb = acc[ni][mi][4 * (g + 1) + j];
              pa[j] = (bf16)va; pb[j] = (bf16)vb;
            }
            uint2 ua = __builtin_bit_cast(uint2, pa), ub = __builtin_bit_cast(uint2, pb);
            auto s0 = __builtin_amdgcn_permlane32_swap(ua.x, ub.x, false, false);
            auto s1 = __builtin_amdgcn_permlane32_swap(ua.y, ub.y, false, false);
            *reinterpret_cast<uint4*>(strip + l31 * ROWB + (nn * 32 + 8 * (g + half)) * 2) = make_uint4(s0[0], s1[0], s0[1], s1[1]);
          }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int it = 0; it < 4; ++it) {  // 8 rows x 128 B per wave-instruction
          const uint4 v = *reinterpret_cast<const uint4*>(strip + (it * 8 + (lane >> 3)) * ROWB + (lane & 7) * 16);
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_s, v), c16_srd, c16_lane + (uint32_t)((it * 8 + mi * 32) * p.ldc) * 2u, 0,
                                                 STP == 2 ? 2 : (STP == 1 ? 16 : 0));
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      drain = 16;
    } else if (A_MODE == 0 && CH == 1 && MI * 4 == 16 && (p.R != nullptr) != (p.C2 != nullptr)) {
      // bf16 output with EITHER a bf16 operand R of the epilogue (C += R, or C *= act'(R): the MLP's backward, R = the saved pre-activation) OR a
      // second output (C2 = act(C): the training forward's MLP-up).  r06: the generic loop below loads R inside the lane's (row < M, column < N)
      // branch and uses it at once -- read off the ISA, `s_waitcnt vmcnt(0)` behind each of the 16 loads of a tile: sixteen exposed round trips to
      // HBM per tile on the largest launch of the training step (the dgrad of MLP-down x act', 2364 tiles).  Here R and both outputs go through
      // buffer descriptors (rows past M / columns past N: the hardware range check), R runs two 32-row passes ahead of its use and nothing is predicated.
      const int mw = m0 + wm * TM;
      const long long rows_left = (long long)p.M - mw;
      auto span16 = [&](long long ld) -> int {
        const long long b = rows_left > 0 ? rows_left * ld * 2 : 0;
        return b > 0x7fffffffLL ? 0x7fffffff : (int)b;
      };
      typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_s;
      const uint32_t oob = (nw0 + (lane & 7) * 8 + 7 < p.N) ? 0u : 0x80000000u;
      const __amdgpu_buffer_rsrc_t c16_srd =
          __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(p.C) + ((size_t)mw * p.ldc + nw0) * 2, 0, span16(p.ldc), 0x00020000);
      const uint32_t c16_lane = ((uint32_t)((lane >> 3) * p.ldc + (lane & 7) * 8) * 2u) | oob;
      auto transpose = [&](int mi) __attribute__((always_inline)) {
#pragma unroll
        for (int nn = 0; nn < 2; ++nn)
#pragma unroll
          for (int g = 0; g < 4; g += 2) {
            bf16x4 pa, pb;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              pa[j] = (bf16)acc[nn][mi][4 * g + j]; pb[j] = (bf16)acc[nn][mi][4 * (g + 1) + j];
            }
            uint2 ua = __builtin_bit_cast(uint2, pa), ub = __builtin_bit_cast(uint2, pb);
            auto s0 = __builtin_amdgcn_permlane32_swap(ua.x, ub.x, false, false);
            auto s1 = __builtin_amdgcn_permlane32_swap(ua.y, ub.y, false, false);
            *reinterpret_cast<uint4*>(strip + l31 * ROWB + (nn * 32 + 8 * (g + half)) * 2) = make_uint4(s0[0], s1[0], s0[1], s1[1]);
          }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      };
      if (p.R != nullptr) {
        const __amdgpu_buffer_rsrc_t r16_srd = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(reinterpret_cast<const char*>(p.R)) + ((size_t)mw * p.ldr + nw0) * 2, 0, span16(p.ldr), 0x00020000);
        const uint32_t r16_lane = ((uint32_t)((lane >> 3) * p.ldr + (lane & 7) * 8) * 2u) | oob;
        u32x4_s rwin[2][4];
        auto rload = [&](int mi, int w) __attribute__((always_inline)) {
#pragma unroll
          for (int it = 0; it < 4; ++it) rwin[w][it] = __builtin_amdgcn_raw_buffer_load_b128(r16_srd, r16_lane + (uint32_t)((it * 8 + mi * 32) * p.ldr) * 2u, 0, 0);
        };
        rload(0, 0);
        rload(1, 1);
        const int mode = p.res_mode;
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
          transpose(mi);
          u32x4_s v[4];
#pragma unroll
          for (int it = 0; it < 4; ++it) v[it] = *reinterpret_cast<const u32x4_s*>(strip + (it * 8 + (lane >> 3)) * ROWB + (lane & 7) * 16);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int it = 0; it < 4; ++it)
            v[it] = __builtin_bit_cast(u32x4_s, combine_res8(__builtin_bit_cast(bf16x8, v[it]), __builtin_bit_cast(bf16x8, rwin[mi & 1][it]), mode));
          __builtin_amdgcn_sched_barrier(0);
          if (mi + 2 < MI) rload(mi + 2, mi & 1);
#pragma unroll
          for (int it = 0; it < 4; ++it)
            __builtin_amdgcn_raw_buffer_store_b128(v[it], c16_srd, c16_lane + (uint32_t)((it * 8 + mi * 32) * p.ldc) * 2u, 0, STP == 2 ? 2 : (STP == 1 ? 16 : 0));
          __builtin_amdgcn_sched_barrier(0);
        }
        drain = 32;  // 16 loads + 16 stores, all unconditional
      } else {
        const __amdgpu_buffer_rsrc_t c2_srd =
            __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(p.C2) + ((size_t)mw * p.ldc2 + nw0) * 2, 0, span16(p.ldc2), 0x00020000);
        const uint32_t c2_lane = ((uint32_t)((lane >> 3) * p.ldc2 + (lane & 7) * 8) * 2u) | oob;
        const int act2 = p.act2;
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
          transpose(mi);
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const u32x4_s v = *reinterpret_cast<const u32x4_s*>(strip + (it * 8 + (lane >> 3)) * ROWB + (lane & 7) * 16);
            __builtin_amdgcn_raw_buffer_store_b128(v, c16_srd, c16_lane + (uint32_t)((it * 8 + mi * 32) * p.ldc) * 2u, 0, STP == 2 ? 2 : (STP == 1 ? 16 : 0));
            bf16x8 a8 = __builtin_bit_cast(bf16x8, v);
            if (act2 != MMAMD_ACT_NONE) {  // (wave-uniform; the same values as store_act_copy)
#pragma unroll
              for (int j = 0; j < 8; j += 2) {
                const f32x2 in = {(float)a8[j], (float)a8[j + 1]};
                const f32x2 o = act2 == MMAMD_ACT_QUICKGELU ? quick_gelu2(in) : gelu_erf2(in);
                a8[j] = (bf16)o[0]; a8[j + 1] = (bf16)o[1];
              }
            }
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_s, a8), c2_srd, c2_lane + (uint32_t)((it * 8 + mi * 32) * p.ldc2) * 2u, 0, 0);
          }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        drain = 32;  // 32 unconditional stores
      }
    } else {
      drain = 0;
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {  // 64 columns (128 B of bf16) per pass
#pragma unroll
          for (int nn = 0; nn < 2; ++nn)
#pragma unroll
            for (int g = 0; g < 4; g += 2) {
              const int ni = 2 * ch + nn;
              bf16x4 pa, pb;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                float va = acc[ni][mi][4 * g + j], vb = acc[ni][mi][4 * (g + 1) + j];
                  pa[j] = (bf16)va; pb[j] = (bf16)vb;
              }
              uint2 ua = __builtin_bit_cast(uint2, pa), ub = __builtin_bit_cast(uint2, pb);
              auto s0 = __builtin_amdgcn_permlane32_swap(ua.x, ub.x, false, false);
              auto s1 = __builtin_amdgcn_permlane32_swap(ua.y, ub.y, false, false);
              *reinterpret_cast<uint4*>(strip + l31 * ROWB + (nn * 32 + 8 * (g + half)) * 2) = make_uint4(s0[0], s1[0], s0[1], s1[1]);
            }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
          for (int it = 0; it < 4; ++it) {  // 8 rows x 128 B per wave-instruction
            const int row = it * 8 + (lane >> 3), c = lane & 7;
            uint4 v = *reinterpret_cast<const uint4*>(strip + row * ROWB + c * 16);
            const int m = m0 + wm * TM + mi * 32 + row, n = nw0 + ch * 64 + c * 8;
            if (m < p.M && n + 7 < p.N) {
              if (p.R != nullptr) {
                const uint4 rr = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(p.R) + (size_t)m * p.ldr + n);
                bf16x8 a8 = __builtin_bit_cast(bf16x8, v), r8 = __builtin_bit_cast(bf16x8, rr);
                a8 = combine_res8(a8, r8, p.res_mode);
                v = __builtin_bit_cast(uint4, a8);
              }
              store16<STP>(reinterpret_cast<bf16*>(p.C) + (size_t)m * p.ldc + n, v);
              store_act_copy(p, v, m, n);
            }
          }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
    if (!more) break;
    vb = nvb;
    tm = ntm;
    tn = ntn;
  }
}

// ---------------------------------------------------------------------------------------------------------
// GROUPED persistent kernel ("PPG"): the persistent kernel above walking the CONCATENATED tile lists of up to two GEMM problems that
// share the epilogue kind (activation, output type) but not the shapes -- the same projection of the two towers of the dual encoder
// (ViT [50432 x N x 768] and text [19712 x N' x 512] at cfg 2).  One launch instead of two on two streams: the second problem's tiles
// fill the partial last round of the first (a persistent workgroup owns its CU for the whole launch, so a second stream's kernels could
// only run in whatever the first one's tail left over -- in-bench every ViT kernel ran 17-60 % slower than alone and the text tower's
// 24-50 us GEMMs took 150 us on average).  Per tile the problem's fields are (re)loaded from the kernel argument segment (scalar loads);
// K, the leading dimensions, the operand bases and the epilogue pointers all change at a problem boundary, and the first K-tile of the NEXT
// tile -- possibly of the other problem -- is DMA'd behind the last K-tile of the current one exactly as in the single-problem kernel.
struct GemmProblem {
  const bf16* A;
  const bf16* W;
  const float* bias;
  const void* R;
  void* C;
  int M, N, K;
  int lda, ldw, ldr, ldc;
  int tiles_m, tiles_n;
};
struct GemmGroupArgs {
  GemmProblem prob[2];
  int nprob;
  int tile_start[3];  // tile_start[i] = first tile id of problem i; tile_start[nprob] = total
  int stagger;
  // slack-aware start-up stagger (experiment knob 1 = per cent, 0 = off): estimated ticks of one tile of problem 0 / 1; a workgroup whose tile
  // list is shorter than its XCD's longest starts late by a share of the difference, so the chip's epilogue bursts spread without adding makespan
  int slack_pct;
  int tile_ticks[2];
  int order;  // experiment knob 2: walk order of the two problems' tiles inside an XCD's slice (0 = first problem, then second)
  // tile-order group per problem: the workgroups an XCD runs concurrently walk gm row panels x all column tiles, column tile slowest inside a
  // group.  gm = 1 is row-major: ALL column tiles of a row panel run at the same time, in lock-step, so every K-slice of the panel is fetched
  // into the XCD's L2 once -- what a GEMM with FEW column tiles and a LONG K wants (MLP-down: 3 column tiles, a 1.5 MiB panel per 256 rows
  // that no cache level keeps between rounds; r04: HBM bytes per launch 1254 -> ... MB, profiles/r04_pmc_residual_kernel.json)
  int gm[2];
  int cn[2];  // column tiles per chunk, per problem (pick_cn): the chunk is the outermost level of each problem's tile order
};

template <bool OUT_F32, int ACT>
__global__ __launch_bounds__(512) void gemm_bf16_nt_kernel_ppg(const GemmGroupArgs g) {
  constexpr int WM = 2, WN = 4, STP = OUT_F32 ? 0 : 2, RDP = 0;
  constexpr int BM = 256, BN = 256, NW = WM * WN;
  constexpr int TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;
  constexpr int A_BYTES = BM * 128, STAGE = (BM + BN) * 128;
  constexpr int A_INSTR = BM / 8 / NW, B_INSTR = BN / 8 / NW, NDMA = A_INSTR + B_INSTR, NF = NI + MI, NM = NI * MI;
  static_assert(NM >= NDMA && NM >= NF && NW % 4 == 0, "interleave needs one MFMA per DMA piece / fragment read");
  constexpr int CH = TN / 64;  // 128-byte column chunks of a wave tile row in bf16
  extern __shared__ __attribute__((aligned(16))) char smem[];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave - wm * WN;
  const int l31 = lane & 31, half = lane >> 5;

  // Tile walk.  Workgroup b runs on XCD b & 7 and is the (b >> 3)-th of that XCD's `nwx` workgroups.  Every XCD owns a contiguous slice of
  // EACH problem's tile list (an eighth of it: operand panels stay in that XCD's L2) and walks its slice of problem 0 first, then its
  // slice of problem 1 -- so the eight XCDs carry equal WORK, not just equal tile counts (a split of the concatenated list gave the
  // last XCDs only the second problem's shorter tiles: K = 512 against 768, they idled a quarter of the launch).
  const int xcd = (int)blockIdx.x & 7, wl = (int)blockIdx.x >> 3;
  const int nwx = ((int)gridDim.x - xcd + 7) >> 3;
  int xb0, xc0, xb1 = 0, xc1 = 0;  // this XCD's slice [base, base + count) of problem 0 / 1
  {
    const int n0 = g.tile_start[1] - g.tile_start[0], q0 = n0 >> 3, r0 = n0 & 7;
    xc0 = q0 + (xcd < r0 ? 1 : 0);
    xb0 = xcd < r0 ? xcd * (q0 + 1) : r0 * (q0 + 1) + (xcd - r0) * q0;
    if (g.nprob > 1) {
      const int n1 = g.tile_start[2] - g.tile_start[1], q1 = n1 >> 3, r1 = n1 & 7;
      xc1 = q1 + (xcd < r1 ? 1 : 0);
      xb1 = xcd < r1 ? xcd * (q1 + 1) : r1 * (q1 + 1) + (xcd - r1) * q1;
    }
  }
  const int nx = xc0 + xc1;  // tiles of this XCD
  if (wl >= nx) return;      // (whole workgroup: before any barrier)
  // XCD-local tile index -> (problem, tile): the GM-grouped order inside each problem's own tile grid
  auto tile_of = [&](int l, int& sel, int& tm, int& tn) __attribute__((always_inline)) {
    int id;
    if (g.order == 1) {         // experiment: the second problem's tiles first
      sel = l < xc1 ? 1 : 0;
      id = sel ? xb1 + l : xb0 + (l - xc1);
    } else if (g.order == 2 && nwx <= xc0) {  // experiment: one round of the first problem, then the second problem's tiles, then the rest
      sel = (l >= nwx && l < nwx + xc1) ? 1 : 0;
      id = sel ? xb1 + (l - nwx) : xb0 + (l < nwx ? l : l - xc1);
    } else {
      sel = l >= xc0 ? 1 : 0;
      id = sel ? xb1 + (l - xc0) : xb0 + l;
    }
    tile_order_map(id, g.prob[sel].tiles_m, g.prob[sel].tiles_n, g.gm[sel], g.cn[sel], tm, tn);  // (1 <= cn <= tiles_n: launcher)
  };

  // DMA source offsets of this lane (see kernel above for the swizzle): depend on the tile, not on K
  const int sw = (4 * (wave & 3) + (lane >> 4)) & 15;
  const int slot = (lane & 15) ^ sw;
  const int row8 = 2 * (lane >> 4) + (slot >> 3);
  const int chunk = slot & 7;
  auto tile_offsets = [&](const GemmProblem& p, int tm, int tn, uint32_t (&ao)[A_INSTR], uint32_t (&bo)[B_INSTR]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < A_INSTR; ++j) {
      int r = tm * BM + 8 * (wave + NW * j) + row8;
      r = r < p.M ? r : p.M - 1;
      ao[j] = ((uint32_t)r * (uint32_t)p.lda + chunk * 8) * 2u;
    }
#pragma unroll
    for (int j = 0; j < B_INSTR; ++j) {
      int r = tn * BN + 8 * (wave + NW * j) + row8;
      r = r < p.N ? r : p.N - 1;
      bo[j] = ((uint32_t)r * (uint32_t)p.ldw + chunk * 8) * 2u;
    }
  };
  int vb = wl, sel = 0;  // XCD-local tile index of the current tile
  int tm, tn;
  tile_of(vb, sel, tm, tn);
  GemmProblem p = g.prob[sel];  // the CURRENT tile's problem (scalar loads from the kernel argument segment, refreshed per tile)
  const char* Ab = reinterpret_cast<const char*>(p.A);
  const char* Wb = reinterpret_cast<const char*>(p.W);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u32p)smem;
  uint32_t a_off[A_INSTR], b_off[B_INSTR];
  auto issue_piece = [&](int buf, int kt, int i) __attribute__((always_inline)) {
    const uint32_t dst = lds0 + buf * STAGE + (i < A_INSTR ? (wave + NW * i) * 1024 : A_BYTES + (wave + NW * (i - A_INSTR)) * 1024);
    if (i < A_INSTR) dma_piece_s(Ab + (size_t)kt * 128, a_off[i], dst);
    else dma_piece_s(Wb + (size_t)kt * 128, b_off[i - A_INSTR], dst);
  };

  const int hsw = l31 >> 1;
  uint32_t ra[2][4], rb[2][4];
#pragma unroll
  for (int bf = 0; bf < 2; ++bf)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t ro = hsw * 256 + (((((l31 & 1) << 3) | (2 * t + half)) ^ hsw) << 4);
      ra[bf][t] = lds0 + bf * STAGE + (wm * TM) * 128 + ro;
      rb[bf][t] = lds0 + bf * STAGE + A_BYTES + (wn * TN) * 128 + ro;
    }
  typedef __attribute__((address_space(3))) const bf16x8* lds_frag_p;

  f32x16 acc[NI][MI];
  bf16x8 xa0[MI], wb0[NI], xa1[MI], wb1[NI];
  auto load_frags = [&](auto bufc, int t, bf16x8 (&xa)[MI], bf16x8 (&wb)[NI]) {
    constexpr int BF = decltype(bufc)::value;
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) wb[ni] = *reinterpret_cast<lds_frag_p>((uintptr_t)(rb[BF][t] + ni * 32 * 128));
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) xa[mi] = *reinterpret_cast<lds_frag_p>((uintptr_t)(ra[BF][t] + mi * 32 * 128));
  };
  auto mma = [&](bf16x8 (&xa)[MI], bf16x8 (&wb)[NI]) {
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
        acc[ni][mi] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[ni], xa[mi], acc[ni][mi], 0, 0, 0);
  };
  auto mma_one = [&](bf16x8 (&xa)[MI], bf16x8 (&wb)[NI], int i) {
    acc[i / MI][i % MI] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[i / MI], xa[i % MI], acc[i / MI][i % MI], 0, 0, 0);
  };
  // one K-tile out of ring buffer BF; behind the first MFMA group one DMA piece each of (ktsrc -> buffer BF^1)
  auto tile_body = [&](auto bufc, int ktsrc, const bool issue) __attribute__((always_inline)) {
    constexpr int BF = decltype(bufc)::value;
    load_frags(bufc, 0, xa0, wb0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      mma_one(xa1, wb1, i);
      if (issue && i < NDMA) issue_piece(BF ^ 1, ktsrc, i);  // wave-uniform scalar branch
      __builtin_amdgcn_sched_barrier(0);
    }
    load_frags(bufc, 1, xa1, wb1);
    mma(xa0, wb0);
    load_frags(bufc, 2, xa0, wb0);
    mma(xa1, wb1);
    load_frags(bufc, 3, xa1, wb1);
    mma(xa0, wb0);
#pragma unroll
    for (int t = 0; t < 3; ++t) {
      if constexpr (RDP == 0) {         // one read of the next k-step behind each of the first NF MFMAs
#pragma unroll
        for (int i = 0; i < NF; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        if constexpr (NM > NF) __builtin_amdgcn_sched_group_barrier(0x008, NM - NF, 0);
      } else if constexpr (RDP == 1) {  // all NF reads in one burst behind the first MFMA (maximum cover)
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, NF, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, NM - 1, 0);
      } else {                          // two reads behind each of the first NF/2 MFMAs
#pragma unroll
        for (int i = 0; i < NF / 2; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, NM - NF / 2, 0);
      }
    }
  };
  using B0 = std::integral_constant<int, 0>;
  using B1 = std::integral_constant<int, 1>;
  auto sync_tile = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  // First barrier of an output tile (r06).  What must have landed is the tile's first K-tile, DMA'd behind the LAST K-tile of the previous
  // tile -- i.e. BEFORE the previous epilogue's loads and stores.  vmcnt retires in issue order, so waiting until at most `drain` operations
  // are outstanding, with drain = the number of vector-memory instructions the epilogue issued (every one of them an unconditional buffer
  // instruction: the count is exact), covers the DMA without draining the epilogue's stores: the r01-r05 vmcnt(0) here paid the write
  // acknowledgement of the tile's last stores at the head of every tile.  0 = wait for everything (first tile; epilogues with predicated ops).
  int drain = 0;
  auto sync_first = [&]() __attribute__((always_inline)) {
    if (drain == 16) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
    else if (drain == 32) asm volatile("s_waitcnt vmcnt(32)" ::: "memory");
    else if (drain == 63) asm volatile("s_waitcnt vmcnt(63)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };

  int KT = p.K >> 6;  // even (launcher), per problem
  tile_offsets(p, tm, tn, a_off, b_off);
#pragma unroll
  for (int i = 0; i < NDMA; ++i) issue_piece(0, 0, i);
  if (g.slack_pct > 0) {
    // work of workgroup w of this XCD = its tiles of problem 0 and 1 times their estimated tile times (all scalar arithmetic)
    auto work_of = [&](int w) -> long long {
      const int ct = (nx - w + nwx - 1) / nwx;
      const int c0 = w < xc0 ? (xc0 - w + nwx - 1) / nwx : 0;
      return (long long)c0 * g.tile_ticks[0] + (long long)(ct - c0) * g.tile_ticks[1];
    };
    long long wmax = 0;
    for (int w = 0; w < nwx && w < nx; ++w) {
      const long long t = work_of(w);
      wmax = t > wmax ? t : wmax;
    }
    const long long slack = wmax - work_of(wl);
    const long long delay = slack * (((wl * 7) % nwx) + 1) / nwx * g.slack_pct / 100;  // shares 1/nwx .. 1 of the slack, scattered over the workgroups
    if (delay > 0) {
      const long long t0 = __builtin_readcyclecounter();
      while (__builtin_readcyclecounter() - t0 < delay) __builtin_amdgcn_s_sleep(32);
    }
  } else if (g.stagger > 0) {
    const int heavy = nx % nwx;  // this XCD's workgroups 0 .. heavy-1 walk one tile more: they start at once
    if (heavy > 0 && wl >= heavy) {
      const long long delay = (long long)g.stagger * (wl - heavy + 1) / (nwx - heavy);
      const long long t0 = __builtin_readcyclecounter();
      while (__builtin_readcyclecounter() - t0 < delay) __builtin_amdgcn_s_sleep(32);
    }
  }

  while (true) {
    const int m0 = tm * BM, n0 = tn * BN;
    const int nvb = vb + nwx;
    const bool more = nvb < nx;
    int ntm = 0, ntn = 0, nsel = sel;
    const char *Abn = Ab, *Wbn = Wb;
    if (more) {
      tile_of(nvb, nsel, ntm, ntn);
      Abn = reinterpret_cast<const char*>(g.prob[nsel].A);
      Wbn = reinterpret_cast<const char*>(g.prob[nsel].W);
    }
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[ni][mi][r] = 0.f;
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int j = 0; j < 8; ++j) xa1[mi][j] = (bf16)0.f;
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
      for (int j = 0; j < 8; ++j) wb1[ni][j] = (bf16)0.f;

#pragma unroll 1
    for (int kt = 0; kt < KT; kt += 2) {
      if (kt == 0) sync_first();
      else sync_tile();
      tile_body(B0{}, kt + 1, true);
      const bool last = kt + 2 >= KT;
      if (last && more) {  // this tile's loads are all issued: switch the DMA source to the next tile's first K-tile
        // (the offsets are computed HERE, not a tile ahead, and again at the head of the next tile: ~40 VALU instructions per tile buy 8 registers
        // in the K loop and 16 in the epilogue, whose residual-load window they bound)
        tile_offsets(g.prob[nsel], ntm, ntn, a_off, b_off);
        Ab = Abn;  // ... which may belong to the other problem
        Wb = Wbn;
      }
      sync_tile();
      tile_body(B1{}, last ? 0 : kt + 2, !last || more);
    }
    mma(xa1, wb1);  // flush the rotated last k-step

    // ---------------- epilogue (LDS strips in ring buffer 1; buffer 0 is receiving the next tile) ----------------
    // fp32 residual: a ring of RD passes of loads in flight, the first RD issued here (before the bias / barrier / first transpose).
    // Measured (tools/gemm_variant_bench.py --variants 60,61,62,63, r02): depth 1 = 2 (out-proj 100.7 / 100.5 us), depth 3 and 4
    // LOSE (115 / 133 us: 21 spilled registers and more loads queued per CU) -- the residual's latency is not what the fp32
    // epilogue waits for; the default stays 1.
    const int nw0 = n0 + wn * TN;
    const int rrow = lane >> 3, rc = (lane & 7) * 4;  // fp32 read-back: 8 rows x 128 B per wave-instruction
#define MMAMD_EPI_PART 1
#include "gemm_epi_f32.inc"
    if (p.bias != nullptr) {
#pragma unroll
      for (int ni = 0; ni < NI; ++ni)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const int n = n0 + wn * TN + ni * 32 + 4 * half + 8 * g4;
          f32x4 bv = {0.f, 0.f, 0.f, 0.f};
          if (n + 3 < p.N) bv = load4(p.bias + n);
#pragma unroll
          for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[ni][mi][4 * g4 + j] += bv[j];
        }
    }
    if constexpr (ACT == MMAMD_ACT_QUICKGELU || (ACT == MMAMD_ACT_GELU_ERF && !OUT_F32)) {  // (activation + fp32 output: inside the fp32 passes; no model path)
#pragma unroll
      for (int ni = 0; ni < NI; ++ni)
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
          for (int r = 0; r < 16; r += 2) {  // adjacent accumulator registers: the pairs need no moves
            const f32x2 in = {acc[ni][mi][r], acc[ni][mi][r + 1]};
            const f32x2 qg = ACT == MMAMD_ACT_QUICKGELU ? quick_gelu2(in) : gelu_erf2(in);
            acc[ni][mi][r] = qg[0]; acc[ni][mi][r + 1] = qg[1];
          }
    }
    constexpr int ROWB = 144;  // 128-byte strip rows + 16 B pad (conflict-free b128 both ways)
    char* strip = smem + STAGE + wave * (32 * ROWB);
    // (below) __syncthreads(): every wave has finished reading the last K-tile out of ring buffer 1 -- issued inside each branch of the
    // wave- and workgroup-uniform residual test, so that the first residual load and its consumer stay in ONE straight-line region (a value
    // that crosses the join of a uniform branch was spilled to scratch by the register allocator: read off the ISA)
    if constexpr (!OUT_F32) __syncthreads();
    if constexpr (OUT_F32) {
#define MMAMD_EPI_PART 2
#include "gemm_epi_f32.inc"
      drain = has_res ? 63 : 32;  // 32 buffer stores (+ 32 buffer loads: more than the 6-bit counter holds)
    } else if (p.R == nullptr) {
      // bf16 output, no residual (qkv, MLP-up): the same strips, stored through a buffer descriptor (rows past M dropped by the range check,
      // columns past N by bit 31 of the lane's offset) -- 16 unconditional stores per wave, which the next tile's first barrier does not drain
      static_assert(CH == 1, "one 64-column chunk per wave tile");
      const int mw = m0 + wm * TM;
      const long long rows_left = (long long)p.M - mw;
      const long long cb = rows_left > 0 ? rows_left * p.ldc * 2 : 0;
      const __amdgpu_buffer_rsrc_t c16_srd = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(p.C) + ((size_t)mw * p.ldc + nw0) * 2, 0,
                                                                               cb > 0x7fffffffLL ? 0x7fffffff : (int)cb, 0x00020000);
      const uint32_t c16_lane = ((uint32_t)((lane >> 3) * p.ldc + (lane & 7) * 8) * 2u) | ((nw0 + (lane & 7) * 8 + 7 < p.N) ? 0u : 0x80000000u);
      typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_s;
#pragma unroll
      for (int mi = 0; mi < MI; ++mi) {
#pragma unroll
        for (int nn = 0; nn < 2; ++nn)
#pragma unroll
          for (int g4 = 0; g4 < 4; g4 += 2) {
            const int ni = nn;
            bf16x4 pa, pb;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float va = acc[ni][mi][4 * g4 + j], vb2 = acc[ni][mi][4 * (g4 + 1) + j];
              pa[j] = (bf16)va; pb[j] = (bf16)vb2;
            }
            uint2 ua = __builtin_bit_cast(uint2, pa), ub = __builtin_bit_cast(uint2, pb);
            auto s0 = __builtin_amdgcn_permlane32_swap(ua.x, ub.x, false, false);
            auto s1 = __builtin_amdgcn_permlane32_swap(ua.y, ub.y, false, false);
            *reinterpret_cast<uint4*>(strip + l31 * ROWB + (nn * 32 + 8 * (g4 + half)) * 2) = make_uint4(s0[0], s1[0], s0[1], s1[1]);
          }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int it = 0; it < 4; ++it) {  // 8 rows x 128 B per wave-instruction
          const uint4 v = *reinterpret_cast<const uint4*>(strip + (it * 8 + (lane >> 3)) * ROWB + (lane & 7) * 16);
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_s, v), c16_srd, c16_lane + (uint32_t)((it * 8 + mi * 32) * p.ldc) * 2u, 0,
                                                 STP == 2 ? 2 : (STP == 1 ? 16 : 0));
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      drain = MI * 4;
    } else {
      drain = 0;  // (predicated residual loads and stores: not countable)
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {  // 64 columns (128 B of bf16) per pass
#pragma unroll
          for (int nn = 0; nn < 2; ++nn)
#pragma unroll
            for (int g4 = 0; g4 < 4; g4 += 2) {
              const int ni = 2 * ch + nn;
              bf16x4 pa, pb;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                float va = acc[ni][mi][4 * g4 + j], vb2 = acc[ni][mi][4 * (g4 + 1) + j];
                  pa[j] = (bf16)va; pb[j] = (bf16)vb2;
              }
              uint2 ua = __builtin_bit_cast(uint2, pa), ub = __builtin_bit_cast(uint2, pb);
              auto s0 = __builtin_amdgcn_permlane32_swap(ua.x, ub.x, false, false);
              auto s1 = __builtin_amdgcn_permlane32_swap(ua.y, ub.y, false, false);
              *reinterpret_cast<uint4*>(strip + l31 * ROWB + (nn * 32 + 8 * (g4 + half)) * 2) = make_uint4(s0[0], s1[0], s0[1], s1[1]);
            }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
          for (int it = 0; it < 4; ++it) {  // 8 rows x 128 B per wave-instruction
            const int row = it * 8 + (lane >> 3), c = lane & 7;
            uint4 v = *reinterpret_cast<const uint4*>(strip + row * ROWB + c * 16);
            const int m = m0 + wm * TM + mi * 32 + row, n = nw0 + ch * 64 + c * 8;
            if (m < p.M && n + 7 < p.N) {
              if (p.R != nullptr) {
                const uint4 rr = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(p.R) + (size_t)m * p.ldr + n);
                bf16x8 a8 = __builtin_bit_cast(bf16x8, v), r8 = __builtin_bit_cast(bf16x8, rr);
#pragma unroll
                for (int j = 0; j < 8; ++j) a8[j] = (bf16)((float)a8[j] + (float)r8[j]);
                v = __builtin_bit_cast(uint4, a8);
              }
              store16<STP>(reinterpret_cast<bf16*>(p.C) + (size_t)m * p.ldc + n, v);
            }
          }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
    if (!more) break;
    vb = nvb;
    tm = ntm;
    tn = ntn;
    if (nsel != sel) {  // wave-uniform: the walk crossed into the next problem
      sel = nsel;
      p = g.prob[sel];
    }
    KT = p.K >> 6;
    tile_offsets(p, tm, tn, a_off, b_off);  // (the values the last K-tile already computed: recomputed so that they are dead across the epilogue)
  }
}


#ifdef MMAMD_EXPERIMENTS
#include "experiments/gemm_kernel_w.inc"  // two-workgroups-per-CU experiment (slower: DESIGN.md 4.1)
#endif

// plain one-thread-per-output kernel: on-device cross-check for the MFMA kernels (tests / debugging)
template <bool OUT_F32>
__global__ __launch_bounds__(256) void gemm_naive_kernel(const GemmArgs p) {
  const int n = blockIdx.x * 64 + (threadIdx.x & 63);
  const int m = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (m >= p.M || n >= p.N) return;
  float acc = 0.f;
  for (int k = 0; k < p.K; ++k) acc = fmaf((float)p.A[(size_t)m * p.lda + k], (float)p.W[(size_t)n * p.ldw + k], acc);
  if (p.bias) acc += p.bias[n];
  acc = apply_act(acc, p.act);
  if constexpr (OUT_F32) {
    if (p.R) acc += reinterpret_cast<const float*>(p.R)[(size_t)m * p.ldr + n];
    reinterpret_cast<float*>(p.C)[(size_t)m * p.ldc + n] = acc;
  } else {
    if (p.R) acc += (float)reinterpret_cast<const bf16*>(p.R)[(size_t)m * p.ldr + n];
    reinterpret_cast<bf16*>(p.C)[(size_t)m * p.ldc + n] = (bf16)acc;
    if (p.C2) reinterpret_cast<bf16*>(p.C2)[(size_t)m * p.ldc2 + n] = (bf16)apply_act((float)(bf16)acc, p.act2);
  }
}

template <int BM, int BN, int WM, int WN, bool OUT_F32, int ACT, bool SGB>
static int launch_tiled(GemmArgs& p, hipStream_t st) {
  constexpr int smem = 2 * (BM + BN) * 128;
  auto kern = gemm_bf16_nt_kernel<BM, BN, WM, WN, OUT_F32, ACT, SGB>;
  static unsigned long long attr_mask = 0;  // per-device one-time opt-in to > 64 KiB dynamic LDS
  if (int rc_attr = opt_in_lds(reinterpret_cast<const void*>(kern), smem, attr_mask)) return rc_attr;
  const int tiles_m = (p.M + BM - 1) / BM;
  p.tiles_n = (p.N + BN - 1) / BN;
  hipLaunchKernelGGL(kern, dim3(tiles_m * p.tiles_n), dim3(WM * WN * 64), smem, st, p);
  return launch_status("gemm_bf16");
}

template <int BM, int BN, int WM, int WN, bool OUT_F32, int ACT, int GM, int ABL = 0, bool LDSEPI = true>
static int launch_tiled_p(GemmArgs& p, hipStream_t st) {
  // the pipelined kernel walks the K-tiles in pairs (compile-time buffer index): odd tile counts take the plain kernel
  if (((p.K >> 6) & 1) != 0) return launch_tiled<BM, BN, WM, WN, OUT_F32, ACT, true>(p, st);
  constexpr int smem = 2 * (BM + BN) * 128;
  auto kern = gemm_bf16_nt_kernel_p<BM, BN, WM, WN, OUT_F32, ACT, GM, ABL, LDSEPI, false, 0>;
  static unsigned long long attr_mask = 0;  // per-device one-time opt-in to > 64 KiB dynamic LDS
  if (int rc_attr = opt_in_lds(reinterpret_cast<const void*>(kern), smem, attr_mask)) return rc_attr;
  const int tiles_m = (p.M + BM - 1) / BM;
  p.tiles_n = (p.N + BN - 1) / BN;
  hipLaunchKernelGGL(kern, dim3(tiles_m * p.tiles_n), dim3(WM * WN * 64), smem, st, p, tiles_m,
                     (ABL & 64) != 0 ? g_gemm_trace : nullptr);
  return launch_status("gemm_bf16_p");
}

#ifdef MMAMD_EXPERIMENTS
#include "experiments/gemm_launchers.inc"
#endif

template <bool OUT_F32, int ACT, int GM, int WM = 2, int WN = 4, int STP = 0, int RDP = 0, int RES_DEPTH = 1, bool BLDS = false, int A_MODE = 0,
          bool BDIR = false>
static int launch_tiled_pp(GemmArgs& p, hipStream_t st) {
  if constexpr (A_MODE == 0) {
    if (((p.K >> 6) & 1) != 0) return launch_tiled<256, 256, 2, 4, OUT_F32, ACT, true>(p, st);
  }
  if constexpr (BDIR) {
    if (p.Wp == nullptr) { set_error("gemm: the direct-W kernel needs the packed weights (mmamd_pack_w_frag)"); return MMAMD_E_BADARG; }
  }
  constexpr int smem = 2 * 512 * 128 + (BLDS ? 1024 : 0);  // + the tile's bias values
  auto kern = gemm_bf16_nt_kernel_pp<OUT_F32, ACT, GM, WM, WN, STP, RDP, RES_DEPTH, BLDS, A_MODE, BDIR>;
  static unsigned long long attr_mask = 0;  // per-device one-time opt-in to > 64 KiB dynamic LDS
  if (int rc_attr = opt_in_lds(reinterpret_cast<const void*>(kern), smem, attr_mask)) return rc_attr;
  const int tiles_m = (p.M + 255) / 256;
  p.tiles_n = (p.N + 255) / 256;
  const int ntiles = tiles_m * p.tiles_n;
  const int cus = stream_cus(st);                   // 256, or the CU partition of a masked stream (multiple of 8: whole XCD slices)
  const int grid = ntiles < cus ? ntiles : cus;  // one persistent workgroup per CU
  p.gm = pick_gm(p.tiles_n, cus);
  p.cn = pick_cn(p.tiles_n, p.K);
  hipLaunchKernelGGL(kern, dim3(grid), dim3(WM * WN * 64), smem, st, p, tiles_m, ntiles);
  return launch_status("gemm_bf16_pp");
}

template <bool OUT_F32, int ACT>
static int launch_grouped(GemmGroupArgs& g, hipStream_t st) {
  constexpr int smem = 2 * 512 * 128;
  auto kern = gemm_bf16_nt_kernel_ppg<OUT_F32, ACT>;
  static unsigned long long attr_mask = 0;  // per-device one-time opt-in to > 64 KiB dynamic LDS
  if (int rc_attr = opt_in_lds(reinterpret_cast<const void*>(kern), smem, attr_mask)) return rc_attr;
  const int ntiles = g.tile_start[g.nprob];
  const int cus = stream_cus(st);
  for (int i = 0; i < 2; ++i) { g.gm[i] = pick_gm(g.prob[i].tiles_n, cus); g.cn[i] = pick_cn(g.prob[i].tiles_n, g.prob[i].K); }
  const int grid = ntiles < cus ? ntiles : cus;  // one persistent workgroup per CU
  hipLaunchKernelGGL(kern, dim3(grid), dim3(512), smem, st, g);
  return launch_status("gemm_bf16_grouped");
}


template <bool OUT_F32, int ACT>
static int dispatch_variant(GemmArgs& p, hipStream_t st) {
  int v = g_gemm_variant;
  if (v == 0) {
    // Default policy (measured per shape with tools/kernel_bench.py):
    //  * the pipelined 256x256 kernel whenever its grid reaches a good fraction of the 256 CUs, else 128x128 tiles;
    //  * wave quantisation: one workgroup per CU, so a grid of r = tiles/256 rounds with a small fractional part pays a
    //    whole extra round (N = 768 GEMMs at B = 256: 591 tiles = 2.31 rounds -> 3).  Then the row range is split: the
    //    first floor(r) full rounds run on 256x256 tiles, the remaining rows on 128x128 tiles (4x the workgroups, ~1/4
    //    the time each), as a second launch on the same stream.
    const int tiles_n = (p.N + 255) / 256, tiles_m = (p.M + 255) / 256;
    const long t256 = (long)tiles_m * tiles_n;
    const int cus = stream_cus(st);              // CU partition of a masked stream, else 256
    const long t_eq = t256 * kChipCUs / cus;     // tile count scaled to a whole chip: the thresholds below were measured on 256 CUs
    // row-range split for the wave-quantisation tail: returns true when it launched (rc holds the status)
    int rc = 0;
    auto try_split = [&](bool big_pp) -> bool {
      const long full = t256 / cus, rem = t256 - full * cus;
      if (!(full >= 1 && full <= 4 && rem > 0 && rem <= cus / 2)) return false;
      const int m_tiles_big = (int)((full * cus) / tiles_n);  // whole row-panels that fit in the full rounds
      if (!(m_tiles_big >= 1 && m_tiles_big < tiles_m)) return false;
      GemmArgs a = p, b = p;
      const size_t rows = (size_t)m_tiles_big * 256;
      a.M = (int)rows;
      b.M = p.M - (int)rows;
      b.A = p.A + rows * p.lda;
      const size_t esz = OUT_F32 ? 4 : 2;
      b.C = reinterpret_cast<char*>(p.C) + rows * p.ldc * esz;
      if (p.R != nullptr) b.R = reinterpret_cast<const char*>(p.R) + rows * p.ldr * esz;
      if (p.C2 != nullptr) b.C2 = reinterpret_cast<char*>(p.C2) + rows * p.ldc2 * 2;
      rc = big_pp ? launch_tiled_pp<OUT_F32, ACT, 8, 2, 4, OUT_F32 ? 0 : 2>(a, st) : launch_tiled_p<256, 256, 2, 4, OUT_F32, ACT, 8>(a, st);
      if (rc == 0) rc = launch_tiled<128, 128, 2, 2, OUT_F32, ACT, true>(b, st);
      return true;
    };
    // (re-measured with warm clocks, tools/kernel_bench.py: the persistent kernel wins from ~400 tiles up at every K — out-proj 625 vs 616 vs
    //  602 TF/s for PP / P / P + split, text MLP-up 691 / 663 / 620, patch embedding 863 / 851 / 838 — and the row-range split only pays
    //  with long K: MLP-down 891 with it, 836-838 without)
    // (half a round of 256 x 256 tiles with a long K: four times as many 128 x 128 tiles balance better -- [9856 x 768 x 3072], the text MLP-down
    //  of FLAVA / CoCa at B = 128, 117 tiles: 55 us vs 63; profiles/r02_gemm_flava_coca_shapes.txt)
    if (t_eq < 96 || (t_eq < 128 && p.K >= 2048)) {
      v = 6;
    } else if ((p.K & 127) == 0 && t_eq >= 400) {
      v = 18;  // many tiles per CU: the persistent kernel hides each tile's first-stage load behind the previous epilogue
      if (p.K >= 2048 && try_split(true)) return rc;
      // the large-M and the small-M launches get different instantiations (tile-order group 8 / 4: equal speed), so that a kernel name in a
      // rocprof summary is ONE shape class — the bench's dominant kernel, gemm_bf16_nt_kernel_pp<false, QuickGELU, 8, ...>, is the ViT MLP-up only
      if (p.M < 32768) return launch_tiled_pp<OUT_F32, ACT, 4, 2, 4, OUT_F32 ? 0 : 2>(p, st);
    } else {
      v = 7;
      if (p.K >= 2048 && try_split(false)) return rc;
    }
  }
  switch (v) {
    case 1: return launch_tiled<256, 256, 2, 4, OUT_F32, ACT, false>(p, st);
    case 2: return launch_tiled<128, 128, 2, 2, OUT_F32, ACT, false>(p, st);
    case 5: return launch_tiled<256, 256, 2, 4, OUT_F32, ACT, true>(p, st);
    case 6: return launch_tiled<128, 128, 2, 2, OUT_F32, ACT, true>(p, st);
    case 7: return launch_tiled_p<256, 256, 2, 4, OUT_F32, ACT, 8>(p, st);
    // bf16 C tiles are stored non-temporal (measured +6-7 % on the qkv / MLP-up GEMMs: the 128 KiB a block writes per
    // tile no longer competes with the operand panels for the XCD's L2); the in-place fp32 residual update stays plain
    case 18: return launch_tiled_pp<OUT_F32, ACT, 8, 2, 4, OUT_F32 ? 0 : 2>(p, st);
    case 70: return launch_tiled_pp<OUT_F32, ACT, 8, 2, 4, OUT_F32 ? 0 : 2, 0, 1, true>(p, st);  // bias through LDS (DMA'd during the K loop)
#ifdef MMAMD_EXPERIMENTS
#include "experiments/gemm_dispatch_cases.inc"
#endif
    default: set_error("gemm: unknown variant %d (experimental variants need -DMMAMD_EXPERIMENTS)", v); return MMAMD_E_BADARG;
  }
}

template <bool OUT_F32>
static int dispatch(GemmArgs& p, hipStream_t st) {
  if (g_gemm_variant == 99) {
    hipLaunchKernelGGL((gemm_naive_kernel<OUT_F32>), dim3((p.N + 63) / 64, (p.M + 3) / 4), dim3(256), 0, st, p);
    return launch_status("gemm_naive");
  }
  switch (p.act) {
    case MMAMD_ACT_NONE: return dispatch_variant<OUT_F32, MMAMD_ACT_NONE>(p, st);
    case MMAMD_ACT_QUICKGELU: return dispatch_variant<OUT_F32, MMAMD_ACT_QUICKGELU>(p, st);
    default: return dispatch_variant<OUT_F32, MMAMD_ACT_GELU_ERF>(p, st);
  }
}

}  // namespace mmamd

using namespace mmamd;

extern "C" int mmamd_set_gemm_variant(int variant) {
  g_gemm_variant = variant;
  return 0;
}
extern "C" int mmamd_get_gemm_variant(void) { return g_gemm_variant; }
extern "C" int mmamd_debug_set_gemm_stagger(int percent) {
  g_gemm_stagger = percent < 0 ? 0 : percent;
  return 0;
}

// host-side enumeration of the persistent kernels' tile order for a tiles_m x tiles_n grid (gm / cn <= 0: the launchers' own choice for contraction length K):
// out[2 * id] = tm, out[2 * id + 1] = tn for id = 0 .. tiles_m * tiles_n - 1.  No device work.
extern "C" int mmamd_debug_tile_order(int tiles_m, int tiles_n, int K, int gm, int cn, int* out) {
  MMAMD_CHECK_ARG(tiles_m > 0 && tiles_n > 0 && K > 0 && out != nullptr, MMAMD_E_BADARG, "debug_tile_order: bad argument");
  if (gm <= 0) gm = pick_gm(tiles_n, 256);
  if (cn <= 0) cn = pick_cn(tiles_n, K);
  cn = cn < tiles_n ? cn : tiles_n;
  for (int id = 0; id < tiles_m * tiles_n; ++id) tile_order_map(id, tiles_m, tiles_n, gm, cn, out[2 * id], out[2 * id + 1]);
  return cn;
}
extern "C" int mmamd_debug_set_gemm_knob(int knob, int value) {
  MMAMD_CHECK_ARG(knob >= 0 && knob < 8, MMAMD_E_BADARG, "debug_set_gemm_knob: knob %d out of range", knob);
  g_gemm_knob[knob] = value;
  if (knob == 5) set_rowln_ablation(value);  // gemm_rowln.hip: timing ablations of the out-projection + LayerNorm kernel
  return 0;
}

extern "C" int mmamd_debug_set_gemm_wp(const void* wp) {
  g_gemm_wp = wp;
  return 0;
}

// W [N, K] bf16 row-major -> MFMA-fragment order (GemmArgs::Wp): ceil(N / 32) x (K / 16) blocks of 64 lanes x 16 B; rows past N are zeros
namespace mmamd {
__global__ __launch_bounds__(256) void pack_w_frag_kernel(const bf16* __restrict__ W, int ldw, int N, int K, bf16* __restrict__ Wp) {
  const int KS = K >> 4;
  const long long total = (long long)((N + 31) >> 5) * KS * 64;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const int lane = (int)(i & 63);
    const long long blk = i >> 6;
    const int ks = (int)(blk % KS), nb = (int)(blk / KS);
    const int n = nb * 32 + (lane & 31), k = ks * 16 + (lane >> 5) * 8;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (n < N) v = *reinterpret_cast<const uint4*>(W + (size_t)n * ldw + k);
    *reinterpret_cast<uint4*>(Wp + i * 8) = v;
  }
}
}  // namespace mmamd

extern "C" int mmamd_pack_w_frag(const void* W, int ldw, int N, int K, void* Wp, mmamd_stream_t stream) {
  MMAMD_CHECK_ARG(W && Wp && N > 0 && K > 0, MMAMD_E_BADARG, "pack_w_frag: bad argument");
  MMAMD_CHECK_ARG(K % 16 == 0 && ldw >= K && ldw % 8 == 0, MMAMD_E_UNSUPPORTED, "pack_w_frag: K=%d must be a multiple of 16, ldw a multiple of 8", K);
  MMAMD_CHECK_ARG(aligned16(W) && aligned16(Wp), MMAMD_E_ALIGN, "pack_w_frag: pointers must be 16-byte aligned");
  const long long total = (long long)((N + 31) / 32) * (K / 16) * 64;
  const unsigned grid = (unsigned)((total + 255) / 256 < 8192 ? (total + 255) / 256 : 8192);
  hipLaunchKernelGGL(pack_w_frag_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, (const bf16*)W, ldw, N, K, (bf16*)Wp);
  return launch_status("pack_w_frag");
}

extern "C" int mmamd_debug_set_gemm_trace(void* buf) {
  g_gemm_trace = reinterpret_cast<unsigned long long*>(buf);
  return 0;
}

static int gemm_bf16_impl(const void* A, int lda, const void* W, int ldw, const float* bias, const void* residual, int ldr, void* C,
                          int ldc, int out_dtype, int M, int N, int K, int act, void* C2, int ldc2, int act2, mmamd_stream_t stream);

extern "C" int mmamd_gemm_bf16(const void* A, int lda, const void* W, int ldw, const float* bias, const void* residual,
                               int ldr, void* C, int ldc, int out_dtype, int M, int N, int K, int act,
                               mmamd_stream_t stream) {
  return gemm_bf16_impl(A, lda, W, ldw, bias, residual, ldr, C, ldc, out_dtype, M, N, K, act, nullptr, 0, 0, stream);
}

extern "C" int mmamd_patch_embed_gemm(const void* image, const void* W, int ldw, const float* pos, float* x, int B, int patch, int image_size,
                                      int width, mmamd_stream_t stream) {
  MMAMD_CHECK_ARG(image && W && pos && x && B >= 0 && width > 0, MMAMD_E_BADARG, "patch_embed_gemm: bad argument");
  MMAMD_CHECK_ARG((patch == 16 || patch == 32) && image_size > 0 && image_size % patch == 0 && image_size % 8 == 0, MMAMD_E_UNSUPPORTED,
                  "patch_embed_gemm: patch %d / image %d (16- and 32-pixel patches of an image side that is a multiple of 8)", patch, image_size);
  MMAMD_CHECK_ARG(width % 8 == 0 && ldw >= 3 * patch * patch && ldw % 8 == 0, MMAMD_E_UNSUPPORTED, "patch_embed_gemm: width %d / ldw %d", width, ldw);
  MMAMD_CHECK_ARG(aligned16(image) && aligned16(W) && aligned16(pos) && aligned16(x), MMAMD_E_ALIGN, "patch_embed_gemm: pointers must be 16-byte aligned");
  const int g = image_size / patch;
  MMAMD_CHECK_ARG((uint64_t)B * 3u * image_size * image_size * 2u < (1ull << 32) && (uint64_t)width * ldw * 2u < (1ull << 32), MMAMD_E_UNSUPPORTED,
                  "patch_embed_gemm: operand exceeds the 4 GiB 32-bit DMA offset range");
  if (B == 0) return 0;
  GemmArgs p;
  p.A = (const bf16*)image; p.W = (const bf16*)W; p.bias = nullptr; p.R = pos; p.C = x;
  p.M = B * g * g; p.N = width; p.K = 3 * patch * patch; p.lda = p.K; p.ldw = ldw; p.ldr = width; p.ldc = width; p.act = MMAMD_ACT_NONE; p.tiles_n = 0;
  p.kt_chunk = 0; p.c_split_stride = 0; p.res_mode = 0; p.C2 = nullptr; p.ldc2 = 0; p.act2 = 0; p.split_flat = 0; p.stagger = 0;
  p.i2c_g2 = g * g; p.i2c_g = g; p.i2c_p = patch; p.i2c_hw = image_size;
  p.i2c_lcr = patch == 16 ? 1 : 2; p.i2c_ltpc = patch == 16 ? 2 : 4; p.i2c_rpk = 64 / patch;
  return launch_tiled_pp<true, MMAMD_ACT_NONE, 8, 2, 4, 0, 0, 1, false, 1>(p, (hipStream_t)stream);
}

extern "C" int mmamd_gemm_bf16_grouped(const mmamd_gemm_problem* probs, int nprob, int out_dtype, int act, mmamd_stream_t stream) {
  MMAMD_CHECK_ARG(probs != nullptr && nprob >= 1 && nprob <= 2, MMAMD_E_BADARG, "gemm_grouped: 1 or 2 problems, got %d", nprob);
  MMAMD_CHECK_ARG(out_dtype == MMAMD_F32 || out_dtype == MMAMD_BF16, MMAMD_E_BADARG, "gemm_grouped: bad out_dtype %d", out_dtype);
  MMAMD_CHECK_ARG(act == MMAMD_ACT_NONE || act == MMAMD_ACT_QUICKGELU || act == MMAMD_ACT_GELU_ERF, MMAMD_E_BADARG, "gemm_grouped: bad activation code %d", act);
  // one persistent launch needs every problem on the persistent kernel's K granularity (two 64-deep K-tiles per loop trip) and enough tiles
  // in total to give each CU more than one; anything else runs as the separate launches the grouped call stands for (same results: a tile's
  // arithmetic does not depend on which launch computes it -- tests/test_gpu_grouped_gemm.py)
  bool group = nprob == 2 && g_gemm_variant == 0;
  long tiles = 0;
  for (int i = 0; i < nprob; ++i) {
    const mmamd_gemm_problem& q = probs[i];
    MMAMD_CHECK_ARG(q.M >= 0 && q.N > 0 && q.K > 0 && q.W && (q.M == 0 || (q.A && q.C)), MMAMD_E_BADARG, "gemm_grouped: problem %d: bad argument", i);
    if ((q.K & 127) != 0 || q.M == 0) group = false;
    tiles += (long)((q.M + 255) / 256) * ((q.N + 255) / 256);
  }
  hipStream_t st = (hipStream_t)stream;
  if (!group || tiles < 2L * stream_cus(st)) {
    for (int i = 0; i < nprob; ++i) {
      const mmamd_gemm_problem& q = probs[i];
      if (q.M == 0) continue;  // an empty problem (its pointers may be NULL)
      if (int rc = gemm_bf16_impl(q.A, q.lda, q.W, q.ldw, q.bias, q.R, q.ldr, q.C, q.ldc, out_dtype, q.M, q.N, q.K, act, nullptr, 0, 0, stream)) return rc;
    }
    return 0;
  }
  GemmGroupArgs g;
  g.nprob = nprob;
  g.tile_start[0] = 0;
  for (int i = 0; i < nprob; ++i) {
    const mmamd_gemm_problem& q = probs[i];
    MMAMD_CHECK_ARG(q.N % 8 == 0, MMAMD_E_UNSUPPORTED, "gemm_grouped: N=%d must be a multiple of 8", q.N);
    MMAMD_CHECK_ARG(q.lda >= q.K && q.ldw >= q.K && q.ldc >= q.N && (!q.R || q.ldr >= q.N), MMAMD_E_BADARG, "gemm_grouped: leading dimension too small");
    MMAMD_CHECK_ARG(q.lda % 8 == 0 && q.ldw % 8 == 0 && q.ldc % 8 == 0 && (!q.R || q.ldr % 8 == 0), MMAMD_E_ALIGN,
                    "gemm_grouped: leading dimensions must be multiples of 8 elements");
    MMAMD_CHECK_ARG(aligned16(q.A) && aligned16(q.W) && aligned16(q.C) && aligned16(q.R) && aligned16(q.bias), MMAMD_E_ALIGN,
                    "gemm_grouped: base pointers must be 16-byte aligned");
    MMAMD_CHECK_ARG((uint64_t)q.M * (uint64_t)q.lda * 2u < (1ull << 32) && (uint64_t)q.N * (uint64_t)q.ldw * 2u < (1ull << 32),
                    MMAMD_E_UNSUPPORTED, "gemm_grouped: operand exceeds the 4 GiB 32-bit DMA offset range");
    GemmProblem& d = g.prob[i];
    d.A = (const bf16*)q.A; d.W = (const bf16*)q.W; d.bias = q.bias; d.R = q.R; d.C = q.C;
    d.M = q.M; d.N = q.N; d.K = q.K; d.lda = q.lda; d.ldw = q.ldw; d.ldr = q.ldr; d.ldc = q.ldc;
    d.tiles_m = (q.M + 255) / 256; d.tiles_n = (q.N + 255) / 256;
    g.tile_start[i + 1] = g.tile_start[i] + d.tiles_m * d.tiles_n;
  }
  for (int i = nprob; i < 2; ++i) { g.prob[i] = g.prob[0]; g.tile_start[i + 1] = g.tile_start[nprob]; }
  {
    const long long t_epi = (out_dtype == MMAMD_F32 ? 27000 : 8000) + (act != MMAMD_ACT_NONE ? 8000 : 0);
    const long long t_tile = (long long)(probs[0].K / 64) * 3500 + t_epi;
    g.stagger = (int)(t_tile * (g_gemm_stagger % 1000) / 100);
    g.slack_pct = g_gemm_knob[1];
    g.order = g_gemm_knob[2];
    for (int i = 0; i < 2; ++i) g.tile_ticks[i] = (int)((long long)(g.prob[i].K / 64) * 3500 + t_epi);
  }
  if (out_dtype == MMAMD_F32) {
    switch (act) {
      case MMAMD_ACT_NONE: return launch_grouped<true, MMAMD_ACT_NONE>(g, st);
      case MMAMD_ACT_QUICKGELU: return launch_grouped<true, MMAMD_ACT_QUICKGELU>(g, st);
      default: return launch_grouped<true, MMAMD_ACT_GELU_ERF>(g, st);
    }
  }
  switch (act) {
    case MMAMD_ACT_NONE: return launch_grouped<false, MMAMD_ACT_NONE>(g, st);
    case MMAMD_ACT_QUICKGELU: return launch_grouped<false, MMAMD_ACT_QUICKGELU>(g, st);
    default: return launch_grouped<false, MMAMD_ACT_GELU_ERF>(g, st);
  }
}

extern "C" int mmamd_gemm_bf16_dual(const void* A, int lda, const void* W, int ldw, const float* bias, void* U, int ldu, void* G,
                                    int ldg, int M, int N, int K, int act, mmamd_stream_t stream) {
  MMAMD_CHECK_ARG(U && G, MMAMD_E_BADARG, "gemm_dual: null output");
  MMAMD_CHECK_ARG(act == MMAMD_ACT_QUICKGELU || act == MMAMD_ACT_GELU_ERF, MMAMD_E_BADARG, "gemm_dual: bad activation code %d", act);
  MMAMD_CHECK_ARG(ldg >= N && ldg % 8 == 0 && aligned16(G), MMAMD_E_ALIGN, "gemm_dual: second output must be 16-byte aligned with ldg %% 8 == 0");
  return gemm_bf16_impl(A, lda, W, ldw, bias, nullptr, 0, U, ldu, MMAMD_BF16, M, N, K, MMAMD_ACT_NONE, G, ldg, act, stream);
}

static int gemm_bf16_impl(const void* A, int lda, const void* W, int ldw, const float* bias, const void* residual, int ldr, void* C,
                          int ldc, int out_dtype, int M, int N, int K, int act, void* C2, int ldc2, int act2, mmamd_stream_t stream) {
  MMAMD_CHECK_ARG(A && W && C, MMAMD_E_BADARG, "gemm: null pointer");
  MMAMD_CHECK_ARG(M >= 0 && N > 0 && K > 0, MMAMD_E_BADARG, "gemm: bad sizes M=%d N=%d K=%d", M, N, K);
  MMAMD_CHECK_ARG(K % 64 == 0, MMAMD_E_UNSUPPORTED, "gemm: K=%d must be a multiple of 64 (pad the operands)", K);
  MMAMD_CHECK_ARG(N % 8 == 0, MMAMD_E_UNSUPPORTED, "gemm: N=%d must be a multiple of 8", N);
  MMAMD_CHECK_ARG(lda >= K && ldw >= K && ldc >= N && (!residual || ldr >= N), MMAMD_E_BADARG, "gemm: leading dimension too small");
  MMAMD_CHECK_ARG(lda % 8 == 0 && ldw % 8 == 0 && ldc % 8 == 0 && (!residual || ldr % 8 == 0), MMAMD_E_ALIGN,
                  "gemm: leading dimensions must be multiples of 8 elements");
  MMAMD_CHECK_ARG(aligned16(A) && aligned16(W) && aligned16(C) && aligned16(residual) && aligned16(bias), MMAMD_E_ALIGN,
                  "gemm: base pointers must be 16-byte aligned");
  MMAMD_CHECK_ARG((uint64_t)M * (uint64_t)lda * 2u < (1ull << 32) && (uint64_t)N * (uint64_t)ldw * 2u < (1ull << 32),
                  MMAMD_E_UNSUPPORTED, "gemm: operand exceeds the 4 GiB 32-bit DMA offset range");
  MMAMD_CHECK_ARG(act >= MMAMD_ACT_NONE && act <= MMAMD_ACT_MUL_GELU_GRAD, MMAMD_E_BADARG, "gemm: bad activation code %d", act);
  if (M == 0) return 0;
  GemmArgs p;
  p.A = (const bf16*)A; p.W = (const bf16*)W; p.bias = bias; p.R = residual; p.C = C;
  p.M = M; p.N = N; p.K = K; p.lda = lda; p.ldw = ldw; p.ldr = ldr; p.ldc = ldc; p.act = act; p.tiles_n = 0;
  p.kt_chunk = 0; p.c_split_stride = 0; p.res_mode = 0;
  p.C2 = C2; p.ldc2 = ldc2; p.act2 = act2; p.split_flat = 0;
  p.Wp = (const bf16*)g_gemm_wp;
  {
    // start-up stagger of the persistent kernel as a fraction (g_gemm_stagger, per cent) of the estimated tile time in shader ticks:
    // ~3500 ticks per 64-deep K-tile + the epilogue (bf16 tile ~8k, + QuickGELU / erf-GELU ~8k, fp32 + residual ~27k)
    const long long t_tile = (long long)(K / 64) * 3500 + (out_dtype == MMAMD_F32 ? 27000 : 8000) +
                             ((act == MMAMD_ACT_QUICKGELU || act == MMAMD_ACT_GELU_ERF) ? 8000 : 0);
    p.stagger = g_gemm_stagger >= 1000 ? -(int)(t_tile * (g_gemm_stagger - 1000) / 100) : (int)(t_tile * g_gemm_stagger / 100);
  }
  if (act == MMAMD_ACT_MUL_QUICKGELU_GRAD || act == MMAMD_ACT_MUL_GELU_GRAD) {
    MMAMD_CHECK_ARG(out_dtype == MMAMD_BF16 && residual != nullptr, MMAMD_E_BADARG,
                    "gemm: the activation-gradient epilogue needs bf16 output and the saved pre-activation as `residual`");
    p.res_mode = act == MMAMD_ACT_MUL_QUICKGELU_GRAD ? 1 : 2;
    p.act = MMAMD_ACT_NONE;
  }
  hipStream_t st = (hipStream_t)stream;
  if (out_dtype == MMAMD_F32) return dispatch<true>(p, st);
  if (out_dtype == MMAMD_BF16) return dispatch<false>(p, st);
  MMAMD_CHECK_ARG(false, MMAMD_E_BADARG, "gemm: bad out_dtype %d", out_dtype);
}

// column-wise sum of `splits` partial outputs (second stage of the split-K weight-gradient GEMM)
namespace mmamd {
__global__ __launch_bounds__(256) void splitk_reduce_kernel(const float* __restrict__ part, int splits, long long n, float* __restrict__ out,
                                                            const float* __restrict__ part2, long long n2, float* __restrict__ out2) {
  // elements [0, n): the weight-gradient partials (split stride n); [n, n + n2): the bias-gradient partials of the CS kernels (split stride n2)
  long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  long long stride = n;
  if (i >= n) {
    i -= n;
    if (i >= n2) return;
    part = part2; out = out2; stride = n2;
  }
  f32x4 acc = load4(part + i);
  for (int s = 1; s < splits; ++s) {
    const f32x4 v = load4(part + (size_t)s * stride + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] += v[j];
  }
  store4(out + i, acc);
}
}  // namespace mmamd

// FLAT (default): 1-D grid of tiles * splits, split-major after the XCD-contiguous remap — an XCD then runs neighbouring tiles of ONE split,
// which stream the same contraction rows at the same time and share operand panels in its L2 (the 2-D grid scattered a split's tiles over all
// XCDs: PMC FETCH_SIZE 3x the operand bytes on the MLP-up gradient).  Measured (tools/wgrad_bench.py --sched): -3...-10 % on every shape.
template <bool TNM, int SCH = 0, int GMV = 8, bool FLAT = true, bool CSK = false>
static int gemm_splitk_impl(const void* A, int lda, const void* W, int ldw, float* C, float* ws, int M, int N, int K, int splits,
                            mmamd_stream_t stream, float* db = nullptr) {
  const int KT = K / 64;
  int chunk = (KT + splits - 1) / splits;
  chunk += chunk & 1;  // even number of K-tiles per split (the K loop is unrolled by two); KT is even, so is the remainder
  const int nsplit = (KT + chunk - 1) / chunk;
  GemmArgs p;
  p.A = (const bf16*)A; p.W = (const bf16*)W; p.bias = nullptr; p.R = nullptr; p.C = nsplit == 1 ? C : ws;
  p.M = M; p.N = N; p.K = K; p.lda = lda; p.ldw = ldw; p.ldr = 0; p.ldc = N; p.act = MMAMD_ACT_NONE;
  p.kt_chunk = chunk; p.c_split_stride = (long long)M * N; p.res_mode = 0;
  p.C2 = nullptr; p.ldc2 = 0; p.act2 = 0; p.split_flat = FLAT ? 1 : 0;
  float* db_part = CSK ? (nsplit == 1 ? db : ws + (size_t)nsplit * M * N) : nullptr;  // bias-gradient partials behind the weight-gradient ones
  p.cs_out = db_part;
  constexpr int smem = 2 * 512 * 128;
  auto kern = gemm_bf16_nt_kernel_p<256, 256, 2, 4, true, MMAMD_ACT_NONE, GMV, 0, true, TNM, SCH, CSK>;
  static unsigned long long attr_mask = 0;  // per-device one-time opt-in to > 64 KiB dynamic LDS
  if (int rc_attr = opt_in_lds(reinterpret_cast<const void*>(kern), smem, attr_mask)) return rc_attr;
  const int tiles_m = (M + 255) / 256;
  p.tiles_n = (N + 255) / 256;
  hipStream_t st = (hipStream_t)stream;
  if (FLAT) hipLaunchKernelGGL(kern, dim3(tiles_m * p.tiles_n * nsplit), dim3(512), smem, st, p, tiles_m, nullptr);
  else hipLaunchKernelGGL(kern, dim3(tiles_m * p.tiles_n, nsplit), dim3(512), smem, st, p, tiles_m, nullptr);
  if (nsplit > 1) {
    const long long n = (long long)M * N;
    const long long n2 = CSK ? (long long)M : 0;  // (n % 4 == 0 and M % 8 == 0: the two ranges never share a 4-element group)
    hipLaunchKernelGGL(splitk_reduce_kernel, dim3((unsigned)(((n + n2) / 4 + 255) / 256)), dim3(256), 0, st, ws, nsplit, n, C, db_part, n2, db);
  }
  return launch_status("gemm_bf16_splitk");
}

// One validation for every TN split-K launcher (single, + column sums, grouped: ADVICE r05 -- they had drifted apart, 2^31 here and 2^32 there).
// dW[M, N] = A[K, M]^T . W[K, N] with A = dY and W = X row-major over the contraction: 64 contraction rows of either operand must stay inside the
// DMA's signed 32-bit byte offsets; M * N % 4 == 0 (from M % 8) is what lets the reduce kernel run in 4-element groups without the weight-gradient
// and the bias-gradient ranges sharing one.
static int tn_splitk_check(const char* who, const void* A, int lda, const void* W, int ldw, const void* C, const void* ws, int M, int N, int K) {
  MMAMD_CHECK_ARG(A && W && C && M > 0 && N > 0 && K > 0, MMAMD_E_BADARG, "%s: bad argument", who);
  MMAMD_CHECK_ARG(K % 128 == 0, MMAMD_E_UNSUPPORTED, "%s: contraction length K=%d must be a multiple of 128", who, K);
  MMAMD_CHECK_ARG(M % 8 == 0 && N % 8 == 0, MMAMD_E_UNSUPPORTED, "%s: M=%d and N=%d must be multiples of 8", who, M, N);
  MMAMD_CHECK_ARG(lda >= M && ldw >= N && lda % 8 == 0 && ldw % 8 == 0, MMAMD_E_BADARG, "%s: bad leading dimension", who);
  MMAMD_CHECK_ARG(aligned16(A) && aligned16(W) && aligned16(C) && aligned16(ws), MMAMD_E_ALIGN, "%s: base pointers must be 16-byte aligned", who);
  MMAMD_CHECK_ARG((uint64_t)64 * (uint64_t)lda * 2u < (1ull << 31) && (uint64_t)64 * (uint64_t)ldw * 2u < (1ull << 31), MMAMD_E_UNSUPPORTED,
                  "%s: leading dimension too large for the 32-bit DMA offsets", who);
  return 0;
}

// ---- grouped weight gradients: one GEMM launch + one reduce launch for up to 8 problems (gemm_bf16_tn_group_kernel above) ----
namespace mmamd {
struct SplitkReduceJob {
  const float* part;
  float* out;
  const float* part2;
  float* out2;
  long long n, n2;
  int splits;
};
struct SplitkReduceJobs {
  SplitkReduceJob j[kTnGroupMax];
};
// splitk_reduce_kernel per job (blockIdx.y): the same sums in the same order
__global__ __launch_bounds__(256) void splitk_reduce_batched_kernel(const SplitkReduceJobs jobs) {
  const SplitkReduceJob& jb = jobs.j[blockIdx.y];
  const float* part = jb.part;
  float* out = jb.out;
  long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  long long stride = jb.n;
  if (i >= jb.n) {
    i -= jb.n;
    if (i >= jb.n2) return;
    part = jb.part2; out = jb.out2; stride = jb.n2;
  }
  if (jb.splits <= 1) return;  // the GEMM wrote this problem's result itself
  f32x4 acc = load4(part + i);
  for (int s = 1; s < jb.splits; ++s) {
    const f32x4 v = load4(part + (size_t)s * stride + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] += v[j];
  }
  store4(out + i, acc);
}
}  // namespace mmamd

static int tn_group_nsplit(int K, int splits, int* chunk_out) {
  const int KT = K / 64;
  int chunk = (KT + splits - 1) / splits;
  chunk += chunk & 1;  // even number of K-tiles per split, as in gemm_splitk_impl
  *chunk_out = chunk;
  return (KT + chunk - 1) / chunk;
}

extern "C" long long mmamd_gemm_bf16_tn_splitk_group_ws(const mmamd_wgrad_job* jobs, int njobs, int splits) {
  if (!jobs || njobs < 1 || splits < 1) return -1;
  long long total = 4;
  for (int i = 0; i < njobs; ++i) {
    if (jobs[i].K <= 0 || jobs[i].K % 128 != 0) return -1;
    int chunk;
    const int ns = tn_group_nsplit(jobs[i].K, splits, &chunk);
    if (ns > 1) total += (long long)ns * jobs[i].M * jobs[i].N + (jobs[i].db ? (long long)ns * jobs[i].M : 0);
  }
  return total;
}

extern "C" int mmamd_gemm_bf16_tn_splitk_group(const mmamd_wgrad_job* jobs, int njobs, int splits, float* ws, mmamd_stream_t stream) {
  MMAMD_CHECK_ARG(jobs && ws && njobs >= 1 && njobs <= kTnGroupMax && splits >= 1, MMAMD_E_BADARG, "gemm_tn_splitk_group: bad argument (1..%d jobs)", kTnGroupMax);
  GemmTnGroupArgs g;
  SplitkReduceJobs rj;
  bool any_cs = false, any_split = false;
  int wg = 0;
  unsigned max_blocks = 1;
  float* wsp = ws;
  for (int i = 0; i < njobs; ++i) {
    const mmamd_wgrad_job& jb = jobs[i];
    if (int rc = tn_splitk_check("gemm_tn_splitk_group", jb.dy, jb.lddy, jb.x, jb.ldx, jb.dw, ws, jb.M, jb.N, jb.K)) return rc;
    int chunk;
    const int nsplit = tn_group_nsplit(jb.K, splits, &chunk);
    GemmArgs& p = g.p[i];
    p = GemmArgs{};
    float* part = nsplit == 1 ? jb.dw : wsp;
    if (nsplit > 1) wsp += (size_t)nsplit * jb.M * jb.N;
    float* db_part = jb.db ? (nsplit == 1 ? jb.db : wsp) : nullptr;
    if (jb.db && nsplit > 1) wsp += (size_t)nsplit * jb.M;
    p.A = (const bf16*)jb.dy; p.W = (const bf16*)jb.x; p.bias = nullptr; p.R = nullptr; p.C = part;
    p.M = jb.M; p.N = jb.N; p.K = jb.K; p.lda = jb.lddy; p.ldw = jb.ldx; p.ldr = 0; p.ldc = jb.N; p.act = MMAMD_ACT_NONE;
    p.kt_chunk = chunk; p.c_split_stride = (long long)jb.M * jb.N; p.res_mode = 0;
    p.C2 = nullptr; p.ldc2 = 0; p.act2 = 0; p.split_flat = 1;
    p.cs_out = db_part;
    p.tiles_n = (jb.N + 255) / 256;
    g.tiles_m[i] = (jb.M + 255) / 256;
    g.nwg[i] = g.tiles_m[i] * p.tiles_n * nsplit;
    g.wg0[i] = wg;
    wg += (g.nwg[i] + 7) & ~7;
    any_cs |= jb.db != nullptr;
    any_split |= nsplit > 1;
    const long long n = (long long)jb.M * jb.N, n2 = jb.db ? (long long)jb.M : 0;
    rj.j[i] = SplitkReduceJob{part, jb.dw, db_part, jb.db, n, n2, nsplit};
    const unsigned nb = (unsigned)(((n + n2) / 4 + 255) / 256);
    if (nsplit > 1 && nb > max_blocks) max_blocks = nb;
  }
  for (int i = njobs; i < kTnGroupMax; ++i) { g.p[i] = GemmArgs{}; g.wg0[i] = wg; g.nwg[i] = 0; g.tiles_m[i] = 0; rj.j[i] = SplitkReduceJob{nullptr, nullptr, nullptr, nullptr, 0, 0, 0}; }
  g.nprob = njobs;
  constexpr int smem = 2 * 512 * 128;
  hipStream_t st = (hipStream_t)stream;
  static unsigned long long attr_cs = 0, attr_plain = 0;  // per-device one-time opt-in to > 64 KiB dynamic LDS
  if (any_cs) {
    auto kern = gemm_bf16_tn_group_kernel<true>;
    if (int rc_attr = opt_in_lds(reinterpret_cast<const void*>(kern), smem, attr_cs)) return rc_attr;
    hipLaunchKernelGGL(kern, dim3(wg), dim3(512), smem, st, g);
  } else {
    auto kern = gemm_bf16_tn_group_kernel<false>;
    if (int rc_attr = opt_in_lds(reinterpret_cast<const void*>(kern), smem, attr_plain)) return rc_attr;
    hipLaunchKernelGGL(kern, dim3(wg), dim3(512), smem, st, g);
  }
  if (any_split) hipLaunchKernelGGL(splitk_reduce_batched_kernel, dim3(max_blocks, njobs), dim3(256), 0, st, rj);
  return launch_status("gemm_bf16_tn_splitk_group");
}

extern "C" int mmamd_gemm_bf16_splitk(const void* A, int lda, const void* W, int ldw, float* C, float* ws, int M, int N, int K,
                                      int splits, mmamd_stream_t stream) {
  MMAMD_CHECK_ARG(A && W && C && ws && M > 0 && N > 0 && K > 0 && splits >= 1, MMAMD_E_BADARG, "gemm_splitk: bad argument");
  MMAMD_CHECK_ARG(K % 128 == 0, MMAMD_E_UNSUPPORTED, "gemm_splitk: K=%d must be a multiple of 128 (pad the operands)", K);
  MMAMD_CHECK_ARG(N % 8 == 0 && (M * (long long)N) % 4 == 0, MMAMD_E_UNSUPPORTED, "gemm_splitk: N=%d must be a multiple of 8", N);
  MMAMD_CHECK_ARG(lda >= K && ldw >= K && lda % 8 == 0 && ldw % 8 == 0, MMAMD_E_BADARG, "gemm_splitk: bad leading dimension");
  MMAMD_CHECK_ARG(aligned16(A) && aligned16(W) && aligned16(C) && aligned16(ws), MMAMD_E_ALIGN, "gemm_splitk: base pointers must be 16-byte aligned");
  MMAMD_CHECK_ARG((uint64_t)M * (uint64_t)lda * 2u < (1ull << 32) && (uint64_t)N * (uint64_t)ldw * 2u < (1ull << 32),
                  MMAMD_E_UNSUPPORTED, "gemm_splitk: operand exceeds the 4 GiB 32-bit DMA offset range");
  return gemm_splitk_impl<false>(A, lda, W, ldw, C, ws, M, N, K, splits, stream);
}

extern "C" int mmamd_gemm_bf16_tn_splitk(const void* A, int lda, const void* W, int ldw, float* C, float* ws, int M, int N, int K,
                                         int splits, mmamd_stream_t stream) {
  MMAMD_CHECK_ARG(ws && splits >= 1, MMAMD_E_BADARG, "gemm_tn_splitk: bad argument");
  if (int rc = tn_splitk_check("gemm_tn_splitk", A, lda, W, ldw, C, ws, M, N, K)) return rc;
#ifdef MMAMD_EXPERIMENTS  // fragment-read placement experiments of the TN main loop (mmamd_set_gemm_variant(40 .. 43))
  if (g_gemm_variant == 40) return gemm_splitk_impl<true, 0, 8, false>(A, lda, W, ldw, C, ws, M, N, K, splits, stream);  // 2-D grid (split = blockIdx.y)
  if (g_gemm_variant == 41) return gemm_splitk_impl<true, 1, 8, false>(A, lda, W, ldw, C, ws, M, N, K, splits, stream);
  if (g_gemm_variant == 42) return gemm_splitk_impl<true, 2, 8, false>(A, lda, W, ldw, C, ws, M, N, K, splits, stream);
  if (g_gemm_variant == 43) return gemm_splitk_impl<true, 3, 8, false>(A, lda, W, ldw, C, ws, M, N, K, splits, stream);
  if (g_gemm_variant == 44) return gemm_splitk_impl<true, 0, 1, false>(A, lda, W, ldw, C, ws, M, N, K, splits, stream);  // tile order: column tile innermost
  if (g_gemm_variant == 45) return gemm_splitk_impl<true, 0, 2, false>(A, lda, W, ldw, C, ws, M, N, K, splits, stream);
  if (g_gemm_variant == 46) return gemm_splitk_impl<true, 0, 1, true>(A, lda, W, ldw, C, ws, M, N, K, splits, stream);  // flat grid, split-major, column tile innermost
  if (g_gemm_variant == 47) return gemm_splitk_impl<true, 0, 8, true>(A, lda, W, ldw, C, ws, M, N, K, splits, stream);  // flat grid, row tile innermost
#endif
  // (fragment-read placement variants 40-43 differ by less than the run-to-run spread of a 20-launch loop — the same kernel measured 295 and
  //  252 us depending on its position in the loop — and the training step time is unchanged by them: the MFMA-first order stays)
  return gemm_splitk_impl<true>(A, lda, W, ldw, C, ws, M, N, K, splits, stream);
}

// dW = dY^T X AND db = column sums of dY from ONE pass over dY (r05: the colsum passes were 6 % of the training step's
// kernel time and ran at the HBM ceiling -- only fusion removes them).  A = dY [K tokens, M], W = X [K tokens, N]; C [M, N] and db [M] fp32;
// ws: (splits + 1) * M * N + splits * M floats.  Same kernel as mmamd_gemm_bf16_tn_splitk (bit-identical C); the workgroups of column tile 0
// also sum their A fragments (gemm_bf16_nt_kernel_p<.., CS = true>), the split partials of both results are summed by one reduce launch.
extern "C" int mmamd_gemm_bf16_tn_splitk_colsum(const void* A, int lda, const void* W, int ldw, float* C, float* db, float* ws, int M, int N,
                                                int K, int splits, mmamd_stream_t stream) {
  MMAMD_CHECK_ARG(db && ws && splits >= 1 && aligned16(db), MMAMD_E_BADARG, "gemm_tn_splitk_colsum: bad argument");
  if (int rc = tn_splitk_check("gemm_tn_splitk_colsum", A, lda, W, ldw, C, ws, M, N, K)) return rc;
  return gemm_splitk_impl<true, 0, 8, true, true>(A, lda, W, ldw, C, ws, M, N, K, splits, stream, db);
}
