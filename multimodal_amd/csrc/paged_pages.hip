// paged_pages.hip — the pages of a key-value cache: forking rows (with reserving and freeing) and compacting the pool.
//
// A page is free while its count in refcounts is not positive.  Everything that picks pages picks the lowest ones in a fixed order, so that results do
// not depend on the order in which workgroups run; the only atomics are integer additions and minima.
#include "paged.h"

namespace mmamd {

struct ForkParams {
  char* pool;
  const int32_t *table, *lengths, *refs, *parents, *reserve_rows;
  int32_t *new_table, *new_lengths, *new_refs, *shortage;
  int32_t *first, *children, *base, *src, *fresh, *found;  // workspace: two per old row, two per new row, the fresh pages, how many there are and how many copies
  int4* copies;                                            // from page, to page, tokens
  int64_t table_row;
  int old_rows, rows, pages, slots, reserve, fresh_max;
  int64_t page_bytes, block_bytes, row_bytes;
  int blocks;
  FastDiv page;
};

// what a new row takes over and needs
struct RowPlan {
  int parent, n, full, rest, kept, want;  // kept: pages that hold its tokens; want: pages up to its reserved ones
};
__device__ __forceinline__ RowPlan plan_row(const ForkParams& p, int r) {
  RowPlan w;
  const int cap = p.slots * (int)p.page.d;
  const int parent = p.parents[r];
  w.parent = (uint32_t)parent < (uint32_t)p.old_rows ? parent : -1;
  w.n = w.parent < 0 ? 0 : clamp_int(p.lengths[w.parent], 0, cap);
  int more = p.reserve_rows != nullptr ? p.reserve_rows[r] : p.reserve;
  more = clamp_int(more, 0, cap - w.n);
  w.full = (int)div_by(p.page, (uint32_t)w.n);
  w.rest = w.n - w.full * (int)p.page.d;
  w.kept = w.full + (w.rest > 0 ? 1 : 0);
  w.want = (int)div_by(p.page, (uint32_t)w.n + (uint32_t)more + p.page.d - 1u);
  return w;
}

__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  return v;
}
// exclusive scan over the 1024 threads of a workgroup; total in every thread
__device__ __forceinline__ int block_scan(int v, int* lds, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int inc = wave_scan(v, lane);
  __syncthreads();
  if (lane == 63) lds[wave] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    const int x = lds[w];
    before += w < wave ? x : 0;
    all += x;
  }
  total = all;
  return before + inc - v;
}

// Workgroup 0 plans: the lowest child of every parent, the pages each new row needs (numbered over the rows in order), the lowest free pages, the
// copies.  The others copy the counts, which paged_fork_apply_kernel then changes by what the tables gain and lose.  Bound by its chain of dependent loads:
// 5.6 us for 160 rows and 965 pages, 7.5 for 384 rows and 10373 pages.
constexpr int kForkOld = 4096;  // old rows whose children are counted in LDS
__global__ __launch_bounds__(1024) void paged_fork_plan_kernel(const ForkParams p) {
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    for (int i = (blockIdx.x - 1) * 1024 + tid; i < p.pages; i += (gridDim.x - 1) * 1024) p.new_refs[i] = p.refs[i];
    return;
  }
  __shared__ int lds[16];
  __shared__ int near_first[kForkOld], near_children[kForkOld];
  int* const first = p.old_rows <= kForkOld ? near_first : p.first;
  int* const children = p.old_rows <= kForkOld ? near_children : p.children;
  int ahead[4];                                      // counts of the next 4096 pages
  auto look = [&](int i0) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + tid * 4 + k;
      ahead[k] = i < p.pages ? p.refs[i] : 1;
    }
  };
  look(0);
  for (int i = tid; i < p.old_rows; i += 1024) { first[i] = 0x7fffffff; children[i] = 0; }
  __threadfence_block();
  __syncthreads();
  for (int r = tid; r < p.rows; r += 1024) {
    const int parent = p.parents[r];
    if ((uint32_t)parent < (uint32_t)p.old_rows) { atomicMin(&first[parent], r); atomicAdd(&children[parent], 1); }
  }
  __threadfence_block();
  __syncthreads();
  if (p.old_rows <= kForkOld)
    for (int i = tid; i < p.old_rows; i += 1024) p.children[i] = children[i];
  int needed = 0;
  for (int r0 = 0; r0 < p.rows; r0 += 1024) {
    const int r = r0 + tid;
    int need = 0, src = -1;
    if (r < p.rows) {
      const RowPlan w = plan_row(p, r);
      need = w.want > w.kept ? w.want - w.kept : 0;
      if (w.rest > 0) {
        const int id = p.table[w.parent * p.table_row + w.full];
        // (the loads past the first-level cache: for more old rows the minima were made by atomics beyond it)
        if ((uint32_t)id < (uint32_t)p.pages && !(__hip_atomic_load(&first[w.parent], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == r && p.refs[id] == 1)) {
          src = id;
          ++need;
        }
      }
      p.new_lengths[r] = w.n;
    }
    int total;
    const int before = block_scan(need, lds, total);
    if (r < p.rows) { p.base[r] = needed + before; p.src[r] = src; }
    needed += total;
  }
  int found = 0;
  for (int i0 = 0; i0 < p.pages && found < needed; i0 += 4096) {  // (both sides are the same in every thread)
    int c[4], mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      c[k] = ahead[k] <= 0;
      mine += c[k];
    }
    if (i0 + 4096 < p.pages) look(i0 + 4096);
    int total;
    int at = found + block_scan(mine, lds, total);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c[k]) {
        if (at < p.fresh_max) p.fresh[at] = i0 + tid * 4 + k;
        ++at;
      }
    found += total;
  }
  if (found > needed) found = needed;
  __threadfence_block();
  int copies = 0;
  for (int r0 = 0; r0 < p.rows; r0 += 1024) {
    const int r = r0 + tid;
    const bool copy = r < p.rows && p.src[r] >= 0 && p.base[r] < found;
    int total;
    const int at = copies + block_scan(copy, lds, total);
    if (copy) p.copies[at] = make_int4(p.src[r], p.fresh[p.base[r]], plan_row(p, r).rest, 0);
    copies += total;
  }
  if (tid == 0) { p.found[0] = found; p.found[1] = copies; p.shortage[0] = needed - found; }
}

// 1024 16-byte pieces of a copy by one workgroup: four loads a thread in flight, then the stores.  at(i): where piece i lies within a page.  OLD: nobody
// has touched the source lately, it is read past the caches as well (us a call: a large compaction 219 against 228; a fork's pages were just written: 65
// against 49).
template <bool OLD, typename At>
__device__ __forceinline__ void copy_pieces(const char* from, char* to, uint32_t first, uint32_t end, At at) {
  uint4 v[4];
  uint64_t o[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t i = first + k * 256 + threadIdx.x;
    o[k] = at(i < end ? i : end - 1);
    if constexpr (OLD) v[k] = load_past(from + o[k]);
    else v[k] = *reinterpret_cast<const uint4*>(from + o[k]);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (first + k * 256 + threadIdx.x < end) store_past(to + o[k], v[k]);
}

// The first rows * share workgroups move data, `share` of them a copy, which split its pieces evenly: the copies differ in their tokens, so cut into stretches of
// one length they were mostly empty or a second round.  The others write tables: one wave per new row, and one per old row that takes back its references.
// Bound by HBM: 240 MB in 40.7 us behind the plan, 5.9 TB/s; 53 MB in 9.2 us.
__global__ __launch_bounds__(256) void paged_fork_apply_kernel(const ForkParams p, uint32_t share, FastDiv per_copy) {
  const uint32_t copiers = (uint32_t)p.rows * share;
  if (blockIdx.x < copiers) {
    const uint32_t k = div_by(per_copy, blockIdx.x), part = blockIdx.x - k * share;
    const int4 c = p.copies[k];                        // (loaded beside the number of copies; behind it, whatever lay there)
    if ((int)k >= p.found[1]) return;
    const uint32_t per = (uint32_t)(c.z * p.row_bytes / 16), all = per * (uint32_t)p.blocks;  // pieces of a block's tokens, of the copy
    const uint32_t mine = (all + share - 1) / share, end = (part + 1) * mine < all ? (part + 1) * mine : all;
    for (uint32_t first = part * mine; first < end; first += 1024)
      copy_pieces<false>(p.pool + c.x * p.page_bytes, p.pool + c.y * p.page_bytes, first, end, [&](uint32_t x) {
        const uint32_t b = x / per;
        return (uint64_t)b * p.block_bytes + (x - b * per) * 16u;
      });
    return;
  }
  const int found = p.found[0];
  const int lane = threadIdx.x & 63, w = (int)(blockIdx.x - copiers) * 4 + (threadIdx.x >> 6);
  if (w < p.rows) {
    const RowPlan row = plan_row(p, w);
    const int src = p.src[w], base = p.base[w];
    for (int j = lane; j < p.slots; j += 64) {
      int id = -1;
      if (j < row.kept && !(j == row.full && src >= 0)) {
        id = p.table[row.parent * p.table_row + j];
        if ((uint32_t)id >= (uint32_t)p.pages) id = -1;
      } else if (j < row.want || (j == row.full && src >= 0)) {
        const int at = base + (src >= 0 ? j - row.full : j - row.kept);
        if (at < found) {
          id = p.fresh[at];
          atomicAdd(&p.new_refs[id], 1);
        }
      }
      p.new_table[(int64_t)w * p.slots + j] = id;
    }
  } else if (w < p.rows + p.old_rows) {
    const int o = w - p.rows, heirs = p.children[o];
    const int cap = p.slots * (int)p.page.d;
    const int n = clamp_int(p.lengths[o], 0, cap), full = (int)div_by(p.page, (uint32_t)n), rest = n - full * (int)p.page.d;
    for (int j = lane; j < p.slots; j += 64) {
      const int id = p.table[o * p.table_row + j];
      if ((uint32_t)id >= (uint32_t)p.pages) continue;
      int gain = -1;
      if (j < full) gain += heirs;
      else if (j == full && rest > 0 && heirs > 0 && p.refs[id] == 1) gain += 1;
      if (gain != 0) atomicAdd(&p.new_refs[id], gain);
    }
  }
}

struct CompactParams {
  char* pool;
  const int32_t *table, *refs;
  int32_t *new_table, *new_refs, *live;
  int32_t *moves, *counts, *rank;              // workspace: how many pages move, live pages per workgroup, a number per page
  int2* moved;                                 // from page, to page
  int64_t table_row, page_bytes;
  int rows, slots, pages, nblk;
};
constexpr int kCompactPer = 1024;  // pages per workgroup of the first two kernels

__global__ __launch_bounds__(1024) void paged_compact_count_kernel(const CompactParams p) {
  __shared__ int lds[16];
  const int i = blockIdx.x * kCompactPer + threadIdx.x;
  int total;
  block_scan(i < p.pages && p.refs[i] > 0, lds, total);
  if (threadIdx.x == 0) p.counts[blockIdx.x] = total;
}

// With M live pages: the k-th live page from M on moves to the k-th free place before M.  Lists both, and numbers the movers and the places.  ALONE: every
// workgroup counts the whole pool itself, which is one launch less and a few loads a thread for a small pool.
template <bool ALONE>
__global__ __launch_bounds__(1024) void paged_compact_plan_kernel(const CompactParams p) {
  __shared__ int lds[16];
  __shared__ int sums[1];
  const int tid = threadIdx.x, blk = blockIdx.x;
  const int i = blk * kCompactPer + tid;
  const bool live = i < p.pages && p.refs[i] > 0;
  int M = 0, mine = 0;                                 // live pages, and those before this workgroup's
  if constexpr (ALONE) {
    int all = 0, before = 0;
    for (int x = tid; x < p.pages; x += 1024) {
      const int c = p.refs[x] > 0;
      all += c;
      before += x < blk * kCompactPer ? c : 0;
    }
    block_scan(all, lds, M);
    block_scan(before, lds, mine);
  } else {
    for (int b0 = 0; b0 < p.nblk; b0 += 1024) {
      const int b = b0 + tid;
      int total;
      const int ex = block_scan(b < p.nblk ? p.counts[b] : 0, lds, total);
      if (b == blk) sums[0] = M + ex;
      M += total;
    }
    __syncthreads();
    mine = sums[0];
  }
  int total, lowest = 0;                               // lowest: live pages before M
  const int l = mine + block_scan(live, lds, total);   // live pages before page i
  if constexpr (ALONE) {
    int c = 0;
    for (int x = tid; x < M; x += 1024) c += p.refs[x] > 0;
    block_scan(c, lds, lowest);
  } else {
    const int mb = M / kCompactPer;
    for (int b0 = 0; b0 < mb; b0 += 1024) {
      const int b = b0 + tid;
      int t;
      block_scan(b < mb ? p.counts[b] : 0, lds, t);
      lowest += t;
    }
    const int x = mb * kCompactPer + tid;
    int t;
    block_scan(x < M && x < p.pages && p.refs[x] > 0, lds, t);
    lowest += t;
  }
  if (i < p.pages) {
    int rank = 0;
    if (live && i >= M) { rank = l - lowest; p.moved[rank].x = i; }
    else if (!live && i < M) { rank = i - l; p.moved[rank].y = i; }
    p.rank[i] = rank;
  }
  if (blk == 0 && tid == 0) { p.live[0] = M; p.moves[0] = M - lowest; }
}

// The first `copiers` workgroups walk the moved pages in stretches of 1024 pieces, the others rewrite the table and the counts.  Bound by HBM: 1.14 GB in 210 us,
// 5.4 TB/s (a large copy: 4.9); 37 MB in 8.2 us.
__global__ __launch_bounds__(256) void paged_compact_apply_kernel(const CompactParams p, uint32_t pieces, uint32_t stretches, FastDiv per_page, uint32_t copiers) {
  if (blockIdx.x < copiers) {
    uint32_t k = div_by(per_page, blockIdx.x);
    int2 m = p.moved[k];                               // (loaded beside the number of moves; behind it, whatever lay there)
    const uint32_t items = (uint32_t)p.moves[0] * stretches;
    for (uint32_t i = blockIdx.x; i < items;) {
      copy_pieces<true>(p.pool + m.x * p.page_bytes, p.pool + m.y * p.page_bytes, (i - k * stretches) * 1024, pieces, [](uint32_t x) { return (uint64_t)x * 16; });
      i += copiers;
      k = div_by(per_page, i);
      if (i < items) m = p.moved[k];
    }
    return;
  }
  const int M = p.live[0];
  const int64_t step = (int64_t)(gridDim.x - copiers) * 256, first = (int64_t)(blockIdx.x - copiers) * 256 + threadIdx.x;
  for (int64_t i = first; i < (int64_t)p.rows * p.slots; i += step) {
    const int r = (int)(i / p.slots), j = (int)(i - (int64_t)r * p.slots);
    int id = p.table[r * p.table_row + j];
    if ((uint32_t)id >= (uint32_t)p.pages || p.refs[id] <= 0) id = -1;
    else if (id >= M) id = p.moved[p.rank[id]].y;
    p.new_table[i] = id;
  }
  for (int64_t i = first; i < p.pages; i += step) p.new_refs[i] = i >= M ? 0 : p.refs[i] > 0 ? p.refs[i] : p.refs[p.moved[p.rank[i]].x];
}

}  // namespace mmamd

using namespace mmamd;

static int64_t up4(int64_t n) { return (n + 3) & ~3ll; }

// most fresh pages that one call can give
static int64_t fork_fresh(int rows, int slots, int pages) {
  const int64_t n = (int64_t)rows * slots;
  return n < pages ? n : pages;
}

extern "C" int64_t mmamd_paged_fork_workspace(int old_rows, int rows, int slots, int pages) {
  MMAMD_CHECK_ARG(old_rows >= 0 && rows >= 0 && slots >= 1 && pages >= 1, MMAMD_E_BADARG, "mmamd_paged_fork_workspace: rows %d -> %d, slots %d, pages %d", old_rows, rows, slots, pages);
  return 4 * (2 * up4(old_rows) + 2 * up4(rows) + 4 * (int64_t)rows + up4(fork_fresh(rows, slots, pages)) + 4);
}

extern "C" int mmamd_paged_fork(void* pool, int pages, int blocks, int page_size, int64_t row_bytes, const int32_t* table, int64_t table_row, const int32_t* lengths,
                                const int32_t* refcounts, int old_rows, int slots, const int32_t* parents, int rows, const int32_t* reserve_rows, int reserve,
                                int32_t* new_table, int32_t* new_lengths, int32_t* new_refcounts, int32_t* shortage, void* workspace, int64_t workspace_bytes,
                                mmamd_stream_t stream) {
  MMAMD_CHECK_ARG(pages >= 1 && blocks >= 1 && page_size >= 1 && slots >= 1 && old_rows >= 0 && rows >= 0, MMAMD_E_BADARG,
                  "mmamd_paged_fork: pages %d, blocks %d, page size %d, slots %d, rows %d -> %d", pages, blocks, page_size, slots, old_rows, rows);
  MMAMD_CHECK_ARG((int64_t)slots * page_size <= 1 << 30 && (int64_t)rows + old_rows <= 65535 && (int64_t)rows * slots <= 0x7fffffffll && pages <= 0x7fffffff - 65536 && (int64_t)page_size * row_bytes * blocks <= 0x7fffffffll, MMAMD_E_UNSUPPORTED,
                  "mmamd_paged_fork: %d slots of %d tokens, %d rows -> %d", slots, page_size, old_rows, rows);
  MMAMD_CHECK_ARG(pool != nullptr && refcounts != nullptr && new_refcounts != nullptr && shortage != nullptr && workspace != nullptr, MMAMD_E_BADARG, "mmamd_paged_fork: null argument");
  MMAMD_CHECK_ARG((old_rows == 0 || (table != nullptr && lengths != nullptr)) && (rows == 0 || (parents != nullptr && new_table != nullptr && new_lengths != nullptr)), MMAMD_E_BADARG,
                  "mmamd_paged_fork: null argument");
  MMAMD_CHECK_ARG(aligned16(pool) && row_bytes > 0 && row_bytes % 16 == 0, MMAMD_E_ALIGN, "mmamd_paged_fork: the pool must be 16-byte aligned, a token %lld bytes (multiples of 16)", (long long)row_bytes);
  MMAMD_CHECK_ARG(workspace_bytes >= mmamd_paged_fork_workspace(old_rows, rows, slots, pages) && aligned16(workspace), MMAMD_E_BADARG, "mmamd_paged_fork: workspace of %lld bytes is too small",
                  (long long)workspace_bytes);
  ForkParams p;
  p.pool = reinterpret_cast<char*>(pool);
  p.table = table; p.lengths = lengths; p.refs = refcounts; p.parents = parents; p.reserve_rows = reserve_rows;
  p.new_table = new_table; p.new_lengths = new_lengths; p.new_refs = new_refcounts; p.shortage = shortage;
  int32_t* w = reinterpret_cast<int32_t*>(workspace);
  p.first = w; w += up4(old_rows);
  p.children = w; w += up4(old_rows);
  p.base = w; w += up4(rows);
  p.src = w; w += up4(rows);
  p.found = w; w += 4;
  p.copies = reinterpret_cast<int4*>(w); w += 4 * (int64_t)rows;
  p.fresh = w;
  p.fresh_max = (int)fork_fresh(rows, slots, pages);
  p.table_row = table_row;
  p.old_rows = old_rows; p.rows = rows; p.pages = pages; p.slots = slots; p.reserve = reserve;
  p.row_bytes = row_bytes; p.block_bytes = row_bytes * page_size; p.page_bytes = p.block_bytes * blocks; p.blocks = blocks;
  p.page = fast_div((uint32_t)page_size);
  hipStream_t st = (hipStream_t)stream;
  int copiers = (pages + 4095) / 4096;
  if (copiers > 64) copiers = 64;
  paged_fork_plan_kernel<<<1 + copiers, 1024, 0, st>>>(p);
  if (int rc = launch_status("paged_fork plan")) return rc;
  if (rows + old_rows == 0) return 0;
  // workgroups of a copy: four pieces a thread if the page is full, but no more than 4096 in all (two rounds of 8 a CU) for many rows
  int64_t share = (p.page_bytes / 16 + 1023) / 1024;
  const int64_t most = rows > 0 ? (4096 + rows - 1) / rows : 1;
  if (share > most) share = most;
  paged_fork_apply_kernel<<<(unsigned)(rows * share + (rows + old_rows + 3) / 4), 256, 0, st>>>(p, (uint32_t)share, fast_div((uint32_t)share));
  return launch_status("paged_fork");
}

extern "C" int64_t mmamd_paged_compact_workspace(int pages) {
  MMAMD_CHECK_ARG(pages >= 1, MMAMD_E_BADARG, "mmamd_paged_compact_workspace: pages %d", pages);
  return 4 * (4 + up4((pages + kCompactPer - 1) / kCompactPer) + 3 * up4(pages));
}

extern "C" int mmamd_paged_compact(void* pool, int pages, int64_t page_bytes, const int32_t* table, int64_t table_row, int rows, int slots, const int32_t* refcounts,
                                   int32_t* new_table, int32_t* new_refcounts, int32_t* live, void* workspace, int64_t workspace_bytes, mmamd_stream_t stream) {
  MMAMD_CHECK_ARG(pages >= 1 && rows >= 0 && slots >= 1 && page_bytes > 0, MMAMD_E_BADARG, "mmamd_paged_compact: pages %d of %lld bytes, %d rows of %d slots", pages, (long long)page_bytes, rows, slots);
  MMAMD_CHECK_ARG(pages <= 0x7fffffff - 65536 && page_bytes <= 0x7fffffffll && (int64_t)pages * ((page_bytes / 16 + 1023) / 1024) <= 0x7fffffffll, MMAMD_E_UNSUPPORTED,
                  "mmamd_paged_compact: %d pages of %lld bytes", pages, (long long)page_bytes);
  MMAMD_CHECK_ARG(pool != nullptr && refcounts != nullptr && new_refcounts != nullptr && live != nullptr && workspace != nullptr && (rows == 0 || (table != nullptr && new_table != nullptr)),
                  MMAMD_E_BADARG, "mmamd_paged_compact: null argument");
  MMAMD_CHECK_ARG(aligned16(pool) && page_bytes % 16 == 0, MMAMD_E_ALIGN, "mmamd_paged_compact: the pool must be 16-byte aligned, with pages of whole 16-byte pieces");
  MMAMD_CHECK_ARG(workspace_bytes >= mmamd_paged_compact_workspace(pages) && aligned16(workspace), MMAMD_E_BADARG, "mmamd_paged_compact: workspace of %lld bytes is too small", (long long)workspace_bytes);
  CompactParams p;
  p.pool = reinterpret_cast<char*>(pool);
  p.table = table; p.refs = refcounts; p.new_table = new_table; p.new_refs = new_refcounts; p.live = live;
  p.nblk = (pages + kCompactPer - 1) / kCompactPer;
  int32_t* w = reinterpret_cast<int32_t*>(workspace);
  p.moves = w; w += 4;
  p.counts = w; w += up4(p.nblk);
  p.rank = w; w += up4(pages);
  p.moved = reinterpret_cast<int2*>(w);
  p.table_row = table_row; p.page_bytes = page_bytes; p.rows = rows; p.slots = slots; p.pages = pages;
  hipStream_t st = (hipStream_t)stream;
  if (pages <= 16384) {
    paged_compact_plan_kernel<true><<<p.nblk, 1024, 0, st>>>(p);
  } else {
    paged_compact_count_kernel<<<p.nblk, 1024, 0, st>>>(p);
    if (int rc = launch_status("paged_compact count")) return rc;
    paged_compact_plan_kernel<false><<<p.nblk, 1024, 0, st>>>(p);
  }
  if (int rc = launch_status("paged_compact plan")) return rc;
  const uint32_t stretches = (uint32_t)((page_bytes / 16 + 1023) / 1024);
  const int64_t entries = (int64_t)rows * slots > pages ? (int64_t)rows * slots : pages;
  const int64_t copiers = (int64_t)pages * stretches < 2048 ? (int64_t)pages * stretches : 2048, writers = (entries + 255) / 256 < 256 ? (entries + 255) / 256 : 256;
  paged_compact_apply_kernel<<<(unsigned)(copiers + writers), 256, 0, st>>>(p, (uint32_t)(page_bytes / 16), stretches, fast_div(stretches), (uint32_t)copiers);
  return launch_status("paged_compact");
}
