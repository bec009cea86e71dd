// pa_pages.hip -- copying, forking, freeing and compacting the pages of a paged
// cache on gfx950.
//
// State: the cache [L, NB, BS, row] (K and V), block tables [R, MB], context
// lengths [R] and a count per page of the sequences that hold it (0: free).
// Everything stays on the device, so a beam step or a compaction is a few
// launches on the caller's stream with no answer to wait for.
//
//  * The data moves as bytes, 16 a load: HBM-bound, each page read and written
//    once.  A work item is kPiece pieces of one page on one plane (a layer's K
//    or V); a thread has kDepth pieces in flight.  256 pages of 12 layers (201 MB)
//    move in 39.5 us, a compaction's 245 pages (289 MB) in 59, the pages begun by 64
//    forks in 12 layers (75 MB) in 15: 5.1, 4.9 and 5 TB/s read + write, where a copy of
//    1 GB runs at 5.1.  Few pages take a launch (3.4 us).
//  * The bookkeeping is exact and independent of the order in which work-groups
//    run: counts change by integer atomics whose sum is all that matters, and
//    whatever is handed out goes by index (the lowest free page to the first
//    entry that needs one), through prefix sums.  It is bound by its chain of round
//    trips: 5 us for a fork of 8 rows, 3.3 for a compaction of 128 pages, 4 of 1024.
#include "pa_device.hpp"

#include <algorithm>

namespace pa {

constexpr int kPgThreads = 256;
constexpr int kDepth = 4;
constexpr int kPiece = kPgThreads * kDepth;  // 16-byte pieces per work item
static_assert(kPiece <= kMaxPiece, "checked by the host against 32-bit piece indices");
constexpr int kScan = 1024;                  // threads of the allocating work-group

__device__ inline int32_t load_now(const int32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Pieces [first, first + kPiece) of page src of a plane, to page dst.
__device__ inline void copy_item(const PagePool& c, int plane, int64_t src, int64_t dst, int first) {
  const bool second = plane >= c.L;
  const int64_t sb = second ? c.v_sb : c.k_sb, st = second ? c.v_st : c.k_st;
  char* base = second ? c.v + (plane - c.L) * c.v_sl : c.k + plane * c.k_sl;
  const char* from = base + src * sb;
  char* to = base + dst * sb;
  const int pieces = c.BS * c.row16;
  u32x4_t x[kDepth];
  int64_t at[kDepth];
#pragma unroll
  for (int i = 0; i < kDepth; ++i) {
    const int n = first + i * kPgThreads + (int)threadIdx.x;
    at[i] = -1;
    if (n < pieces) {
      const uint32_t row = fastdiv((uint32_t)n, c.row_div);
      at[i] = (int64_t)row * st + (int64_t)(n - (int)row * c.row16) * 16;
      x[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(from + at[i]));
    }
  }
#pragma unroll
  for (int i = 0; i < kDepth; ++i)
    if (at[i] >= 0) __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4_t*>(to + at[i]));
}

__host__ __device__ inline int page_items(const PagePool& c) { return (c.BS * c.row16 + kPiece - 1) / kPiece; }

// ------------------------------------------------------------------- copy --

constexpr int kMaxGrid = 1 << 20;  // work-groups of a launch; the rest is a loop

// A work item is kPiece pieces of one pair's page on one plane.  A destination
// named twice takes the last pair that names it, whichever order the
// work-groups run in.
__global__ __launch_bounds__(kPgThreads) void copy_pages_kernel(const CopyParams p) {
  const uint32_t items = (uint32_t)page_items(p.pool);
  const int64_t all = (int64_t)p.N * p.pool.planes * items;
  for (int64_t x = blockIdx.x; x < all; x += gridDim.x) {
    const int64_t y = x / items;
    const int first = (int)(x - y * items) * kPiece;
    const int i = (int)(y / p.pool.planes), plane = (int)(y - (int64_t)i * p.pool.planes);
    const int32_t src = p.src[i], dst = p.dst[i];
    if (src < 0 || dst < 0 || src >= p.pool.num_blocks || dst >= p.pool.num_blocks || src == dst) continue;
    int again = 0;
    for (int j = i + 1 + (int)threadIdx.x; j < p.N; j += kPgThreads)
      again |= p.dst[j] == dst && p.src[j] >= 0 && p.src[j] < p.pool.num_blocks;
    if (__syncthreads_or(again)) continue;
    copy_item(p.pool, plane, src, dst, first);
  }
}

hipError_t launch_copy_pages(const CopyParams& p, hipStream_t stream) {
  const int64_t all = (int64_t)p.N * p.pool.planes * page_items(p.pool);
  note_launch("pa::copy_pages_kernel");
  hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)std::min<int64_t>(all, kMaxGrid)), dim3(kPgThreads), 0, stream, p);
  return hipGetLastError();
}

// ------------------------------------------------------------------- fork --

// Whether entry i is the first that names its row (a wave's lanes search together).
__device__ inline bool first_of_row(const int32_t* rows, int i, int32_t row) {
  bool again = false;
  for (int j = threadIdx.x & 63; j < i; j += 64) again |= rows[j] == row;
  return __builtin_amdgcn_ballot_w64(again) == 0;
}

// Pages a row holds: those of its context, or none where it exceeds the table.
__device__ inline int pages_of(const ForkParams& p, int32_t len) {
  return len > 0 && (int64_t)len <= (int64_t)p.MB * p.BS ? (int)fastdiv((uint32_t)(len - 1), p.bs_div) + 1 : 0;
}

// One wave's entry: the row's old pages are let go, the parent's whole pages are
// counted once more and its pages kept aside, since another entry may replace the
// parent's own row.  No table changes yet.  Returns the page that the parent has
// begun, or -1.  (Both rows' lengths, then both rows' pages, come in one round trip
// each: a fork of few rows is its chain of round trips.)
__device__ inline int32_t share_entry(const ForkParams& p, int i) {
  const int lane = threadIdx.x & 63;
  const int64_t NB = p.pool.num_blocks;
  const int32_t row = p.rows[i], par = p.parents ? p.parents[i] : -1;
  const bool first = first_of_row(p.rows, i, row);
  if (row < 0 || row >= p.R || !first) {
    if (lane == 0) {
      p.ws_len[i] = -1;
      p.ws_last[i] = -1;
      p.result[i] = kForkInvalid;
    }
    return -1;
  }
  const bool from = par >= 0 && par < p.R;
  const int32_t old_len = p.lens[row], par_len = p.lens[from ? par : row];
  const int32_t* old = p.tables + row * p.tb_stride;
  const int32_t* src = p.tables + (from ? par : row) * p.tb_stride;
  int32_t len = from ? max(par_len, 0) : 0, last = -1, res = par >= p.R ? kForkInvalid : kForkNone;
  const int held = pages_of(p, old_len), n = pages_of(p, len);
  bool bad = len > 0 && n == 0;
  int32_t mine = -1;  // the parent's page number `lane`
  for (int j = lane; j < max(held, n); j += 64) {
    const int32_t pg = j < n ? src[j] : 0, was = j < held ? old[j] : -1;
    if (j < n) p.ws_pages[(int64_t)i * p.MB + j] = pg;
    if (was >= 0 && was < NB) atomicAdd(p.refs + was, -1);
    bad |= j < n && (pg < 0 || pg >= NB);
    mine = j < 64 ? pg : mine;
  }
  if (__builtin_amdgcn_ballot_w64(bad) != 0) {
    len = 0;
    res = kForkInvalid;
  } else {
    const int whole = (int)fastdiv((uint32_t)len, p.bs_div);
    for (int j = lane; j < whole; j += 64) atomicAdd(p.refs + (j < 64 ? mine : src[j]), 1);
    if (whole < n) last = whole < 64 ? __shfl(mine, whole, 64) : src[whole];
  }
  if (lane == 0) {
    p.ws_len[i] = len;
    p.ws_last[i] = last;
    p.result[i] = res;
  }
  return last;
}

__global__ __launch_bounds__(kPgThreads) void fork_share_kernel(const ForkParams p) {
  const int i = blockIdx.x * (kPgThreads / 64) + (threadIdx.x >> 6);
  if (i < p.N) share_entry(p, i);
}

// Exclusive prefix sum over the work-group's kScan threads, and the total.
__device__ inline int scan_block(int v, int& total, int* s_part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();  // (s_part of the last call has been read)
  if (lane == 63) s_part[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kScan / 64; ++w) {
    const int n = s_part[w];
    before += w < wave ? n : 0;
    total += n;
  }
  return before + x - v;
}

// The first pages that nobody holds, as many as `need`: put(rank, page) in ascending
// order, in one pass over the counts that ends when there are enough.  Returns how
// many there were.
template <typename Put>
__device__ inline int find_free(const ForkParams& p, int need, int* s_part, const Put& put) {
  const int64_t NB = p.pool.num_blocks;
  int found = 0;
  for (int64_t b0 = 0; b0 < NB && found < need; b0 += 4 * kScan) {
    int32_t r[4];
    int n = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t pg = b0 + 4 * (int)threadIdx.x + k;
      r[k] = pg < NB ? load_now(p.refs + pg) : 1;
      n += r[k] == 0;
    }
    int total;
    int rank = found + scan_block(n, total, s_part);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (r[k] != 0) continue;
      if (rank < need) put(rank, (int32_t)(b0 + 4 * (int)threadIdx.x + k));
      ++rank;
    }
    found += total;
  }
  return min(found, need);
}

// Pages for the entries, in one work-group.  A begun page that nobody holds any more
// goes to the lowest entry forked from it; every other entry with a begun page gets
// a copy, in the lowest free page, in the order of the entries.
//
// Up to kScan entries, one a thread, compared through LDS (kShare: share_entry() of
// each before, which saves a launch where every wave has one at most).
template <bool kShare>
__global__ __launch_bounds__(kScan) void fork_few_kernel(const ForkParams p) {
  __shared__ int s_part[kScan / 64];
  __shared__ int32_t s_last[kScan], s_free[kScan];
  const int i = threadIdx.x;
  if constexpr (kShare) {
    for (int k = i >> 6; k < p.N; k += kScan / 64) {
      const int32_t last = share_entry(p, k);
      if ((i & 63) == 0) s_last[k] = last;
    }
  } else {
    if (i < p.N) s_last[i] = p.ws_last[i];
  }
  __syncthreads();
  const int32_t last = i < p.N ? s_last[i] : -1;
  bool takes = last >= 0 && load_now(p.refs + last) == 0;
  if (takes) {
    for (int k = 0; k < i; ++k) takes = takes && s_last[k] != last;
  }
  const bool wants = last >= 0 && !takes;
  __syncthreads();  // the counts of begun pages have been read
  if (takes) atomicExch(p.refs + last, 1);
  int need;
  const int rank = scan_block(wants ? 1 : 0, need, s_part);
  const int found = find_free(p, need, s_part, [&](int at, int32_t pg) { s_free[at] = pg; });
  __syncthreads();
  if (i >= p.N) return;
  const int32_t fresh = wants && rank < found ? s_free[rank] : -1;
  p.ws_new[i] = fresh;
  if (fresh >= 0) atomicExch(p.refs + fresh, 1);
  if (wants) p.result[i] = fresh >= 0 ? fresh : kForkNoPage;
}

// The same for any number of entries, compared through ws_owner.
__global__ __launch_bounds__(kScan) void fork_many_kernel(const ForkParams p) {
  __shared__ int s_part[kScan / 64];
  const int tid = threadIdx.x;
  for (int i = tid; i < p.N; i += kScan) {
    const int32_t last = p.ws_last[i];
    if (last >= 0) atomicExch(p.ws_owner + last, INT32_MAX);
  }
  __syncthreads();
  for (int i = tid; i < p.N; i += kScan) {
    const int32_t last = p.ws_last[i];
    if (last >= 0 && load_now(p.refs + last) == 0) atomicMin(p.ws_owner + last, i);
  }
  __syncthreads();
  // Ranks of the entries that need a page, kept in ws_new until it is known.
  int need = 0;
  for (int i0 = 0; i0 < p.N; i0 += kScan) {
    const int i = i0 + tid;
    const int32_t last = i < p.N ? p.ws_last[i] : -1;
    const bool takes = last >= 0 && load_now(p.ws_owner + last) == i;
    const bool wants = last >= 0 && !takes;
    int total;
    const int rank = need + scan_block(wants ? 1 : 0, total, s_part);
    if (i < p.N) p.ws_new[i] = wants ? rank : -1;
    need += total;
  }
  __syncthreads();  // the owners have been read: their pages may be counted
  for (int i = tid; i < p.N; i += kScan) {
    const int32_t last = p.ws_last[i];
    if (last >= 0 && p.ws_new[i] < 0) atomicExch(p.refs + last, 1);
  }
  __syncthreads();
  // ws_owner's use is over: its first entries take the free pages.
  const int found =
      find_free(p, need, s_part, [&](int at, int32_t pg) { atomicExch(p.ws_owner + at, pg); });
  __syncthreads();
  for (int i = tid; i < p.N; i += kScan) {
    const int rank = p.ws_new[i];
    if (rank < 0) continue;
    if (rank < found) {
      const int32_t pg = load_now(p.ws_owner + rank);
      p.ws_new[i] = pg;
      p.result[i] = pg;
      atomicExch(p.refs + pg, 1);
    } else {
      p.ws_new[i] = -1;
      p.result[i] = kForkNoPage;
    }
  }
}

// The first N work-groups write the rows (an entry without a page lets go of
// what it shared and ends empty); the others copy the begun pages.
__global__ __launch_bounds__(kPgThreads) void fork_write_kernel(const ForkParams p) {
  if ((int)blockIdx.x < p.N) {
    const int i = blockIdx.x;
    int32_t len = p.ws_len[i];
    if (len < 0) return;
    const int32_t row = p.rows[i];
    const int32_t* src = p.ws_pages + (int64_t)i * p.MB;
    int32_t* dst = p.tables + row * p.tb_stride;
    const int whole = (int)fastdiv((uint32_t)len, p.bs_div);
    if (p.result[i] == kForkNoPage) {
      for (int j = threadIdx.x; j < whole; j += kPgThreads) atomicAdd(p.refs + src[j], -1);
      len = 0;
    }
    const int n = pages_of(p, len);
    const int32_t fresh = p.ws_new[i];
    for (int j = threadIdx.x; j < p.MB; j += kPgThreads)
      dst[j] = j >= n ? -1 : j == whole && fresh >= 0 ? fresh : src[j];
    if (threadIdx.x == 0) p.lens[row] = len;
    return;
  }
  const uint32_t items = (uint32_t)page_items(p.pool);
  const int64_t all = (int64_t)p.N * p.pool.planes * items;
  for (int64_t x = (int64_t)blockIdx.x - p.N; x < all; x += (int64_t)gridDim.x - p.N) {
    const int64_t y = x / items;
    const int i = (int)(y / p.pool.planes);
    const int32_t fresh = p.ws_len[i] < 0 ? -1 : p.ws_new[i];
    if (fresh >= 0)
      copy_item(p.pool, (int)(y - (int64_t)i * p.pool.planes), p.ws_last[i], fresh, (int)(x - y * items) * kPiece);
  }
}

// Rows emptied without a cache or workspace: one launch.
__global__ __launch_bounds__(kPgThreads) void free_kernel(const ForkParams p) {
  const int i = blockIdx.x * (kPgThreads / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (i >= p.N) return;
  const int32_t row = p.rows[i];
  if (row < 0 || row >= p.R || !first_of_row(p.rows, i, row)) return;
  int32_t* t = p.tables + row * p.tb_stride;
  const int held = pages_of(p, p.lens[row]);
  for (int j = lane; j < p.MB; j += 64) {
    const int32_t pg = t[j];
    if (j < held && pg >= 0 && pg < p.pool.num_blocks) atomicAdd(p.refs + pg, -1);
    t[j] = -1;
  }
  if (lane == 0) p.lens[row] = 0;
}

hipError_t launch_free(const ForkParams& p, hipStream_t stream) {
  note_launch("pa::free_kernel");
  hipLaunchKernelGGL(free_kernel, dim3((unsigned)((p.N + 3) / 4)), dim3(kPgThreads), 0, stream, p);
  return hipGetLastError();
}

// Most entries that the allocating work-group shares itself, a wave each (in two
// launches and in three, tables of 16 pages: 8 entries 8.6 and 10.3 us, 16 entries 8.9
// and 10.3; 32 entries 11.2 both, 64 entries 15.0 and 12.3).
constexpr int kForkFused = kScan / 64;

hipError_t launch_fork(const ForkParams& p, hipStream_t stream) {
  hipError_t e;
  if (p.N <= kForkFused) {
    note_launch("pa::fork_few_kernel<true>");
    hipLaunchKernelGGL(fork_few_kernel<true>, dim3(1), dim3(kScan), 0, stream, p);
  } else {
    note_launch("pa::fork_share_kernel");
    hipLaunchKernelGGL(fork_share_kernel, dim3((unsigned)((p.N + 3) / 4)), dim3(kPgThreads), 0, stream, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (p.N <= kScan) {
      note_launch("pa::fork_few_kernel<false>");
      hipLaunchKernelGGL(fork_few_kernel<false>, dim3(1), dim3(kScan), 0, stream, p);
    } else {
      note_launch("pa::fork_many_kernel");
      hipLaunchKernelGGL(fork_many_kernel, dim3(1), dim3(kScan), 0, stream, p);
    }
  }
  if ((e = hipGetLastError()) != hipSuccess) return e;
  const int64_t copies = std::min<int64_t>((int64_t)p.N * p.pool.planes * page_items(p.pool), kMaxGrid);
  note_launch("pa::fork_write_kernel");
  hipLaunchKernelGGL(fork_write_kernel, dim3((unsigned)(p.N + copies)), dim3(kPgThreads), 0, stream, p);
  return hipGetLastError();
}

// ---------------------------------------------------------------- compact --
// With n live pages, live page q >= n number j (ascending) moves to the free
// page below n number j: as few moves as any dense order needs, and the pages
// written (below n) are never read.

constexpr int kCompactPer = kCompactPages / kPgThreads;  // consecutive pages of a thread

__device__ inline int block_sum(int v, int* s_part) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if (lane == 0) s_part[threadIdx.x >> 6] = v;
  __syncthreads();
  return s_part[0] + s_part[1] + s_part[2] + s_part[3];
}

// Page `pg` of count r: `all` pages live in all, `below` of them before page `all`,
// `before` before this one (moved on).  A moved page's map entry holds its number in
// the order of the moves, as -2 - number, until the move writes where it goes.
__device__ inline void place_page(const CompactParams& p, int pg, int32_t r, int all, int below, int& before) {
  const bool live = r > 0;
  if (pg < all) {
    if (!live) p.ws_to[pg - before] = pg;
    p.page_map[pg] = live ? pg : -1;
  } else {
    if (live) p.ws_from[before - below] = pg;
    p.page_map[pg] = live ? -2 - (before - below) : -1;
  }
  p.refs_out[pg] = r;
  before += live;
}

__global__ __launch_bounds__(kPgThreads) void compact_count_kernel(const CompactParams p) {
  __shared__ int s_part[4];
  int n = 0;
#pragma unroll
  for (int k = 0; k < kCompactPer; ++k) {
    const int64_t pg = (int64_t)blockIdx.x * kCompactPages + k * kPgThreads + threadIdx.x;
    n += pg < p.pool.num_blocks && p.refs[pg] > 0;
  }
  n = block_sum(n, s_part);
  if (threadIdx.x == 0) p.ws_count[blockIdx.x] = n;
}

__global__ __launch_bounds__(kPgThreads) void compact_map_kernel(const CompactParams p) {
  __shared__ int s_part[4];
  const int tid = threadIdx.x;
  const int64_t NB = p.pool.num_blocks;
  // Live pages: in all, before this block, and before page `live` itself (the
  // free pages among the first `live` are as many as the live ones after them).
  int all = 0, mine = 0;
  for (int b = tid; b < p.blocks; b += kPgThreads) {
    const int c = p.ws_count[b];
    all += c;
    mine += b < (int)blockIdx.x ? c : 0;
  }
  all = block_sum(all, s_part);
  mine = block_sum(mine, s_part);
  const int cut = all / kCompactPages;  // the block that holds page `all`
  int below = 0;
  for (int b = tid; b < cut; b += kPgThreads) below += p.ws_count[b];
  for (int k = tid; k < all - cut * kCompactPages; k += kPgThreads)
    below += p.refs[(int64_t)cut * kCompactPages + k] > 0;
  below = block_sum(below, s_part);

  // This block's pages, kCompactPer consecutive ones per thread.
  const int64_t first = (int64_t)blockIdx.x * kCompactPages + tid * kCompactPer;
  int32_t r[kCompactPer];
  int n = 0;
#pragma unroll
  for (int k = 0; k < kCompactPer; ++k) {
    r[k] = first + k < NB ? p.refs[first + k] : 0;
    n += r[k] > 0;
  }
  const int lane = tid & 63;
  int x = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) s_part[tid >> 6] = x;
  __syncthreads();
  int before = mine + x - n;
  for (int w = 0; w < (tid >> 6); ++w) before += s_part[w];
#pragma unroll
  for (int k = 0; k < kCompactPer; ++k) {
    const int64_t pg = first + k;
    if (pg >= NB) break;
    place_page(p, (int)pg, r[k], all, below, before);
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.ws_moves[0] = all - below;
    p.num_live[0] = all;
  }
}

// The same for few pages, in one launch of one work-group: kPlanPer consecutive
// pages of a thread (128 pages 12.9 -> 9.8 us a call).
constexpr int kPlanPer = 8;
constexpr int kPlanPages = kScan * kPlanPer;

__global__ __launch_bounds__(kScan) void compact_plan_kernel(const CompactParams p) {
  __shared__ int s_part[kScan / 64];
  __shared__ int s_below;
  const int NB = (int)p.pool.num_blocks, first = threadIdx.x * kPlanPer;
  int32_t r[kPlanPer];
  int n = 0;
#pragma unroll
  for (int k = 0; k < kPlanPer; ++k) {
    r[k] = first + k < NB ? p.refs[first + k] : 0;
    n += r[k] > 0;
  }
  int all;
  const int start = scan_block(n, all, s_part);
  // Live pages before page `all`.
  if (threadIdx.x == 0) s_below = all;  // (none after it, unless a thread finds it)
  __syncthreads();
  if (all >= first && all < first + kPlanPer) {
    int below = start;
#pragma unroll
    for (int k = 0; k < kPlanPer; ++k) below += first + k < all && r[k] > 0;
    s_below = below;
  }
  __syncthreads();
  const int below = s_below;
  int before = start;
#pragma unroll
  for (int k = 0; k < kPlanPer; ++k) {
    const int pg = first + k;
    if (pg >= NB) break;
    place_page(p, pg, r[k], all, below, before);
  }
  if (threadIdx.x == 0) {
    p.ws_moves[0] = all - below;
    p.num_live[0] = all;
  }
}

// The moves, and the tables brought in line.  A table entry whose page's map
// entry is being written meanwhile reads either form of it: the number leads to
// the same place.
__global__ __launch_bounds__(kPgThreads) void compact_move_kernel(const CompactParams p) {
  const int moves = p.ws_moves[0];
  const int64_t NB = p.pool.num_blocks, step = (int64_t)gridDim.x * kPgThreads;
  const int64_t at = (int64_t)blockIdx.x * kPgThreads + threadIdx.x;
  for (int64_t j = at; j < moves; j += step) {
    const int32_t from = p.ws_from[j], to = p.ws_to[j];
    const int32_t count = p.refs[from];
    p.page_map[from] = to;
    p.refs_out[to] = count;
    p.refs_out[from] = 0;
  }
  for (int64_t e = at; e < (int64_t)p.R * p.MB; e += step) {
    const int64_t row = e / p.MB, col = e - row * p.MB;
    int32_t pg = p.tables[row * p.tb_stride + col];
    if (pg >= 0 && pg < NB) {
      pg = load_now(p.page_map + pg);
      if (pg <= -2) pg = p.ws_to[-2 - pg];
    }
    p.tables_out[row * p.tbo_stride + col] = pg;
  }
  const uint32_t items = (uint32_t)page_items(p.pool);
  const int64_t all = (int64_t)moves * p.pool.planes * items;
  for (int64_t x = blockIdx.x; x < all; x += gridDim.x) {
    const int64_t y = x / items;
    const int j = (int)(y / p.pool.planes);
    copy_item(p.pool, (int)(y - (int64_t)j * p.pool.planes), p.ws_from[j], p.ws_to[j], (int)(x - y * items) * kPiece);
  }
}

hipError_t launch_compact(const CompactParams& p, hipStream_t stream) {
  hipError_t e;
  if (p.pool.num_blocks <= kPlanPages) {
    note_launch("pa::compact_plan_kernel");
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kScan), 0, stream, p);
  } else {
    note_launch("pa::compact_count_kernel");
    hipLaunchKernelGGL(compact_count_kernel, dim3(p.blocks), dim3(kPgThreads), 0, stream, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    note_launch("pa::compact_map_kernel");
    hipLaunchKernelGGL(compact_map_kernel, dim3(p.blocks), dim3(kPgThreads), 0, stream, p);
  }
  if ((e = hipGetLastError()) != hipSuccess) return e;
  // At most half of the pages move.
  const int64_t work = std::max<int64_t>((p.pool.num_blocks / 2 + 1) * p.pool.planes * page_items(p.pool),
                                         (int64_t)p.R * p.MB / kPgThreads + 1);
  note_launch("pa::compact_move_kernel");
  hipLaunchKernelGGL(compact_move_kernel, dim3((unsigned)std::min<int64_t>(work, 2048)), dim3(kPgThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace pa
