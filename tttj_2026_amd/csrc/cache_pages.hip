// Pages of a cache on the device: sequences forked, freed and extended by pages, pages moved to the cache's low end, and
// the copies of pages that both ask for.
//
// The state is a page table [batch, columns], lengths [batch] and uses [pages] (how many rows hold a page, and what holds
// the program has on it otherwise; 0: free).  One block works the new state out, phase by phase, with counters in LDS, and a
// second launch copies; of a large state, each phase is a launch.
#include "cache_checks.hpp"
#include "kernels.hpp"
#include "seq_attention.hpp"

#include <atomic>

namespace tt {

constexpr int kPageThreads = 1024;
constexpr int kPageWaves = kPageThreads / 64;
constexpr int kEach = 4;              // pages that a thread looks at in turn
constexpr int kSmallPages = 16384;    // one block: up to this many pages (8 bytes of LDS each) ...
constexpr int kSmallRows = 512;       // ... and rows (16 bytes each), times their spans of 64 columns
constexpr int kScanBlocks = 256;      // blocks of a launch that counts pages

// Sum over the block's threads before this one; `total` over all.  (s_sums: an int per wave; free again at return.)
__device__ __forceinline__ int block_scan(int v, int* s_sums, int& total) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int upto = wave_scan_int(v);
  if (lane == 63) s_sums[wave] = upto;
  __syncthreads();
  const int sums = wave_scan_int(lane < kPageWaves ? s_sums[lane] : 0);
  total = __builtin_amdgcn_readlane(sums, kPageWaves - 1);
  const int before = wave > 0 ? __builtin_amdgcn_readlane(sums, max(wave - 1, 0)) : 0;
  __syncthreads();
  return before + upto - v;
}

struct PagesArgs {
  const int32_t *table, *lengths, *uses, *parents, *counts;
  int32_t *new_table, *new_lengths, *new_uses;
  int64_t table_row;
  int batch, columns, pages, page_shift, list;  // list: free pages that can be needed
  int *hold, *first, *free_pages;               // large: [pages], [pages], [list]
  int4* rows;                                   // large: [batch]
  int *sums, *needed, *open;                    // large: [kScanBlocks], pages that are needed, and that are free
  int *source, *target, *tokens, *copies;       // copies to make, and their number
};

__device__ __forceinline__ int held_pages(int tokens, int shift) { return (int)(((int64_t)tokens + (1 << shift) - 1) >> shift); }

__device__ __forceinline__ int row_length(const PagesArgs& a, int b) {
  return min(max(a.lengths[b], 0), a.columns << a.page_shift);
}

// What becomes of row b: the row that it continues (or -1), its length, the tokens that it takes over, and the pages that
// row b held.
__device__ __forceinline__ int4 fork_row(const PagesArgs& a, int b) {
  const int p = a.parents == nullptr ? b : a.parents[b];
  const int own = row_length(a, b);
  const int64_t count = a.counts == nullptr ? 0 : a.counts[b];
  if ((uint32_t)p >= (uint32_t)a.batch) return make_int4(-1, 0, 0, held_pages(own, a.page_shift));
  const int before = row_length(a, p);
  const int after = (int)min(max(before + count, (int64_t)0), (int64_t)(a.columns << a.page_shift));
  return make_int4(p, after, min(before, after), held_pages(own, a.page_shift));
}

// Whole pages that a row takes over are shared.  One that it takes over in part is going to be written: of the rows that
// do so the first keeps it, if no row holds it whole and the program has no hold on it; the others get copies.  New pages
// are the lowest free ones, in the order of the rows.
constexpr int kAhead = 4;  // rows whose entries are asked for at once

// Column i of rows b0, b0 + step, ...: `hold` comes to the holds after the call, without the rows as they were and with the
// pages that rows keep whole; `first` to the first row that takes a page over in part.
__device__ __forceinline__ void fork_count(const PagesArgs& a, const int4* rows, int* hold, int* first, int b0, int step,
                                           int i) {
  int had[kAhead], has[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    had[j] = has[j] = -1;
    const int b = b0 + j * step;
    if (b >= a.batch) continue;
    const int4 r = rows[b];
    if (i < r.w) had[j] = a.table[b * a.table_row + i];
    if (i << a.page_shift < r.z) has[j] = a.table[r.x * a.table_row + i];
  }
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    if ((uint32_t)had[j] < (uint32_t)a.pages) atomicAdd(hold + had[j], -1);
    if ((uint32_t)has[j] < (uint32_t)a.pages) {
      const int b = b0 + j * step;
      if ((i + 1) << a.page_shift <= rows[b].z) atomicAdd(hold + has[j], 1);
      else atomicMin(first + has[j], b);
    }
  }
}

// What each row needs and copies, by the whole block: rows become (row that it continues, length, pages taken over, the
// first of its new pages in the list of free ones).
__device__ __forceinline__ void fork_rows(const PagesArgs& a, int4* rows, int* hold, const int* first, int* s_sums,
                                          int& needed, int& copies) {
  const int tid = threadIdx.x, shift = a.page_shift, page = 1 << shift;
  needed = copies = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kPageThreads) {
    const int b = b0 + tid;
    int need = 0, whole = 0, p = -1;
    int4 r = make_int4(-1, 0, 0, 0);
    bool copy = false;
    if (b < a.batch) {
      r = rows[b];
      whole = held_pages(r.z, shift);
      if (r.z & (page - 1)) {
        p = a.table[r.x * a.table_row + whole - 1];
        if ((uint32_t)p < (uint32_t)a.pages) {
          // (only the first row of a page may find it unheld, and it alone changes that)
          if (first[p] == b && hold[p] == 0) hold[p] = 1;
          else copy = true;
        }
      }
      whole -= copy ? 1 : 0;
      need = held_pages(r.y, shift) - whole;
    }
    int total, copied;
    const int begin = needed + block_scan(need, s_sums, total);
    const int at = copies + block_scan(copy ? 1 : 0, s_sums, copied);
    if (b < a.batch) {
      rows[b] = make_int4(r.x, r.y, whole, begin);
      a.new_lengths[b] = r.y;
      if (copy) {
        a.source[at] = p;
        a.tokens[at] = r.z & (page - 1);
        a.target[at] = -1 - b;  // its first new page, once there is one
      }
    }
    needed += total;
    copies += copied;
  }
}

// Free pages among kEach from p0 on of this thread get a rank from `found` on, and the first `take` a hold and a place in
// the list; by the whole block.
__device__ __forceinline__ void fork_list(const PagesArgs& a, const int* hold, int* free_pages, int p0, int end, int take,
                                          int* s_sums, int& found) {
  int held[kEach], open = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int p = p0 + kEach * (int)threadIdx.x + j;
    held[j] = p < end ? hold[p] : 1;
    open += held[j] == 0 ? 1 : 0;
  }
  int total, rank = block_scan(open, s_sums, total) + found;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int p = p0 + kEach * (int)threadIdx.x + j;
    if (p >= end) continue;
    int uses = held[j];
    if (uses == 0) {
      if (rank < take) {
        free_pages[rank] = p;
        uses = 1;
      }
      ++rank;
    }
    a.new_uses[p] = uses;
  }
  found += total;
}

// Column i of rows b0, b0 + step, ... of the new table; `found` free pages are listed.
__device__ __forceinline__ void fork_table(const PagesArgs& a, const int4* rows, const int* free_pages, int found, int b0,
                                           int step, int i) {
  int p[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    p[j] = -1;
    const int b = b0 + j * step;
    if (b >= a.batch) continue;
    const int4 r = rows[b];
    if (i < r.z) {
      p[j] = a.table[r.x * a.table_row + i];
    } else if (i < held_pages(r.y, a.page_shift)) {
      const int rank = r.w + i - r.z;
      if (rank < found) p[j] = free_pages[rank];
    }
  }
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    const int b = b0 + j * step;
    if (b < a.batch) a.new_table[(int64_t)b * a.columns + i] = p[j];
  }
}

__device__ __forceinline__ int copy_target(const int4* rows, const int* free_pages, int found, int row) {
  const int rank = rows[row].w;
  return rank < found ? free_pages[rank] : -1;
}

// One block: each phase needs all that the one before it counted, and a barrier costs less than a launch.  A wave takes a
// row at a time, a lane a column.  Bound by latency: 4.7 us for 4 rows of 35 columns and 90 pages, 9.4 for 128 of 35 and 1493
// (33 with the counters in memory and a thread per entry).
__global__ __launch_bounds__(kPageThreads) void cache_fork_kernel(PagesArgs a) {
  extern __shared__ __align__(16) int pages_lds[];
  __shared__ int s_sums[kPageWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int4* const rows = reinterpret_cast<int4*>(pages_lds);
  int* const hold = pages_lds + 4 * a.batch;
  int* const first = hold + a.pages;
  int* const free_pages = first;  // (which is done with before these are listed)
  for (int b = tid; b < a.batch; b += kPageThreads) rows[b] = fork_row(a, b);
  for (int p = tid; p < a.pages; p += kPageThreads) {
    hold[p] = a.uses[p];
    first[p] = a.batch;
  }
  __syncthreads();
  for (int b0 = wave; b0 < a.batch; b0 += kAhead * kPageWaves)
    for (int i = lane; i < a.columns; i += 64) fork_count(a, rows, hold, first, b0, kPageWaves, i);
  __syncthreads();
  int needed, copies;
  fork_rows(a, rows, hold, first, s_sums, needed, copies);
  __syncthreads();
  const int take = min(needed, a.list);
  int found = 0;
  for (int p0 = 0; p0 < a.pages; p0 += kEach * kPageThreads)
    fork_list(a, hold, free_pages, p0, a.pages, take, s_sums, found);
  found = min(found, take);
  __syncthreads();
  for (int b0 = wave; b0 < a.batch; b0 += kAhead * kPageWaves)
    for (int i = lane; i < a.columns; i += 64) fork_table(a, rows, free_pages, found, b0, kPageWaves, i);
  for (int c = tid; c < copies; c += kPageThreads)  // (barriers lie between)
    a.target[c] = copy_target(rows, free_pages, found,
                              -1 - __hip_atomic_load(a.target + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  if (tid == 0) *a.copies = copies;
}

// The same for large states, a launch per phase: 64 rows of 100 columns 28 us a call at 16385 pages, 28 at 10^6, most of it
// the launches.
__global__ __launch_bounds__(256) void cache_fork_begin_kernel(PagesArgs a) {
  const int step = (int)gridDim.x * 256;
  for (int b = (int)blockIdx.x * 256 + (int)threadIdx.x; b < a.batch; b += step) a.rows[b] = fork_row(a, b);
  for (int p = (int)blockIdx.x * 256 + (int)threadIdx.x; p < a.pages; p += step) {
    a.hold[p] = a.uses[p];
    a.first[p] = a.batch;
  }
}

// Waves take kAhead rows and 64 columns at a time.
template <class F>
__device__ __forceinline__ void each_entry(const PagesArgs& a, F&& f) {
  const int spans = (a.columns + 63) / 64, tasks = (a.batch + kAhead - 1) / kAhead * spans;
  for (int t = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); t < tasks; t += (int)gridDim.x * 4) {
    const int i = t % spans * 64 + (int)(threadIdx.x & 63);
    if (i < a.columns) f(t / spans * kAhead, i);
  }
}

__global__ __launch_bounds__(256) void cache_fork_count_kernel(PagesArgs a) {
  each_entry(a, [&](int b0, int i) { fork_count(a, a.rows, a.hold, a.first, b0, 1, i); });
}

__global__ __launch_bounds__(kPageThreads) void cache_fork_rows_kernel(PagesArgs a) {
  __shared__ int s_sums[kPageWaves];
  int needed, copies;
  fork_rows(a, a.rows, a.hold, a.first, s_sums, needed, copies);
  if (threadIdx.x == 0) *a.needed = needed, *a.copies = copies;
}

// Pages that a block of a launch over all of them looks at.
struct Share {
  int begin, end;
};
__device__ __forceinline__ Share share_of(const PagesArgs& a) {
  const int most = kEach * kPageThreads, turns = (a.pages + most - 1) / most;
  const int each = (turns + (int)gridDim.x - 1) / (int)gridDim.x * most;
  const int begin = (int)min((int64_t)blockIdx.x * each, (int64_t)a.pages);
  return {begin, (int)min((int64_t)begin + each, (int64_t)a.pages)};
}

// sums: how many of each block's pages are free, or for a compaction used.
__global__ __launch_bounds__(kPageThreads) void cache_count_kernel(PagesArgs a, const int* pages, bool used) {
  __shared__ int s_sums[kPageWaves];
  const Share s = share_of(a);
  int n = 0, total;
  for (int p = s.begin + (int)threadIdx.x; p < s.end; p += kPageThreads) n += (used ? pages[p] > 0 : pages[p] == 0) ? 1 : 0;
  block_scan(n, s_sums, total);
  if (threadIdx.x == 0) a.sums[blockIdx.x] = total;
}

// The sum before this block's; `total` of all.
__device__ __forceinline__ int sums_before(const PagesArgs& a, int* s_sums, int& total) {
  static_assert(kScanBlocks <= kPageThreads, "a thread per block");
  const int tid = threadIdx.x, n = tid < (int)gridDim.x ? a.sums[tid] : 0;
  int before;
  block_scan(tid < (int)blockIdx.x ? n : 0, s_sums, before);
  block_scan(n, s_sums, total);
  return before;
}

__global__ __launch_bounds__(kPageThreads) void cache_fork_list_kernel(PagesArgs a) {
  __shared__ int s_sums[kPageWaves];
  const Share s = share_of(a);
  const int take = min(*a.needed, a.list);
  int total, found = sums_before(a, s_sums, total);
  for (int p0 = s.begin; p0 < s.end; p0 += kEach * kPageThreads)
    fork_list(a, a.hold, a.free_pages, p0, s.end, take, s_sums, found);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.open = min(total, take);
}

__global__ __launch_bounds__(256) void cache_fork_table_kernel(PagesArgs a) {
  const int found = *a.open, copies = *a.copies;
  each_entry(a, [&](int b0, int i) { fork_table(a, a.rows, a.free_pages, found, b0, 1, i); });
  for (int c = (int)blockIdx.x * 256 + (int)threadIdx.x; c < copies; c += (int)gridDim.x * 256)
    a.target[c] = copy_target(a.rows, a.free_pages, found, -1 - a.target[c]);
}

// The used pages numbered from their count on move to the free ones below it, both in order: the fewest moves, none of
// which reads what another writes.
__device__ __forceinline__ int compacted(const PagesArgs& a, const int* number, int b, int i, int held) {
  if (i >= held) return -1;
  const int p = a.table[b * a.table_row + i];
  return (uint32_t)p < (uint32_t)a.pages ? number[p] : p;
}

__global__ __launch_bounds__(kPageThreads) void cache_compact_kernel(PagesArgs a) {
  extern __shared__ __align__(16) int pages_lds[];
  __shared__ int s_sums[kPageWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // The number that a page gets; and the pages that move, then where to.
  int* const number = pages_lds;
  int* const movers = pages_lds + a.pages;
  int* const holes = movers + a.pages / 2;
  int used = 0;
  for (int p = tid; p < a.pages; p += kPageThreads) used += a.uses[p] > 0 ? 1 : 0;
  int total;
  block_scan(used, s_sums, total);
  used = total;
  int moving = 0, filling = 0;
  for (int p0 = 0; p0 < a.pages; p0 += kEach * kPageThreads) {
    int uses[kEach], both = 0;  // moves in the upper half, holes in the lower
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int p = p0 + kEach * tid + j;
      uses[j] = p < a.pages ? max(a.uses[p], 0) : 0;
      both += (uses[j] > 0 && p >= used ? 1 << 16 : 0) + (p < used && uses[j] == 0 ? 1 : 0);
    }
    static_assert(kEach * kPageThreads < 1 << 15, "both counts fit");
    const int before = block_scan(both, s_sums, total);
    int r = moving + (before >> 16), s = filling + (before & 0xffff);
    moving += total >> 16;
    filling += total & 0xffff;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int p = p0 + kEach * tid + j;
      if (p >= a.pages) continue;
      const bool moves = uses[j] > 0 && p >= used;
      if (moves) movers[r++] = p;
      else if (p < used && uses[j] == 0) holes[s++] = p;
      number[p] = p;
      if (moves || p >= used) a.new_uses[p] = 0;
      else if (uses[j] > 0) a.new_uses[p] = uses[j];
    }
  }
  __syncthreads();
  for (int r = tid; r < moving; r += kPageThreads) {
    const int p = movers[r], q = holes[r];
    number[p] = q;
    a.new_uses[q] = a.uses[p];
    a.source[r] = p;
    a.target[r] = q;
  }
  __syncthreads();
  for (int b = wave; b < a.batch; b += kPageWaves) {
    const int held = held_pages(row_length(a, b), a.page_shift);
    for (int i = lane; i < a.columns; i += 64) a.new_table[(int64_t)b * a.columns + i] = compacted(a, number, b, i, held);
  }
  if (tid == 0) *a.copies = moving;
}

// Large: with u of the U used pages below page p, p is hole number p - u, or of the pages that move the one with U - 1 - u
// behind it; so the sums of used pages are all that blocks need of one another.  (hold: pages that move, the last first,
// and in its upper half the holes.  first: the numbers that pages get.)
__global__ __launch_bounds__(kPageThreads) void cache_compact_list_kernel(PagesArgs a) {
  __shared__ int s_sums[kPageWaves];
  const Share s = share_of(a);
  int used, below = sums_before(a, s_sums, used);
  for (int p0 = s.begin; p0 < s.end; p0 += kEach * kPageThreads) {
    int uses[kEach], n = 0, total;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int p = p0 + kEach * (int)threadIdx.x + j;
      uses[j] = p < s.end ? max(a.uses[p], 0) : 0;
      n += uses[j] > 0 ? 1 : 0;
    }
    int u = below + block_scan(n, s_sums, total);
    below += total;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int p = p0 + kEach * (int)threadIdx.x + j;
      if (p >= s.end) continue;
      if (p == used) *a.copies = used - u;
      a.first[p] = p;
      if (p >= used) {
        if (uses[j] > 0) a.hold[used - 1 - u] = p;
        a.new_uses[p] = 0;
      } else if (uses[j] == 0) {
        a.hold[a.pages / 2 + p - u] = p;
      } else {
        a.new_uses[p] = uses[j];
      }
      u += uses[j] > 0 ? 1 : 0;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0 && used == a.pages) *a.copies = 0;
}

__global__ __launch_bounds__(256) void cache_compact_moves_kernel(PagesArgs a) {
  const int moving = *a.copies;
  for (int r = (int)blockIdx.x * 256 + (int)threadIdx.x; r < moving; r += (int)gridDim.x * 256) {
    const int p = a.hold[moving - 1 - r], q = a.hold[a.pages / 2 + r];
    a.first[p] = q;
    a.new_uses[q] = a.uses[p];
    a.source[r] = p;
    a.target[r] = q;
  }
}

__global__ __launch_bounds__(256) void cache_compact_table_kernel(PagesArgs a) {
  each_entry(a, [&](int b0, int i) {
    for (int b = b0; b < min(b0 + kAhead, a.batch); ++b)
      a.new_table[(int64_t)b * a.columns + i] = compacted(a, a.first, b, i, held_pages(row_length(a, b), a.page_shift));
  });
}

// One block, with `lds` bytes for the counters.
template <class K>
static int launch_pages(const char* what, K kernel, int lds, const PagesArgs& a, std::atomic<uint64_t>& ready,
                        hipStream_t stream) {
  int dev = 0;
  TT_HIP(hipGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if ((ready.load(std::memory_order_relaxed) & bit) == 0) {
    TT_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                               16 * kSmallRows + 8 * kSmallPages));
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  hipLaunchKernelGGL(kernel, dim3(1), dim3(kPageThreads), lds, stream, a);
  return launch_status(what);
}

// One block's phases against a launch for each, us a call of a fork (in a graph) and of a compaction: 64 rows of 64 columns 16
// to 30 (18 to 24) and 14 to 23 at 500 pages, 16 to 28 (18 to 30) and 19 to 25 at 16384; 512 of 64 20 to 30 (24 to 24) and 15 to
// 24 at 500 pages, 27 to 29 (31 to 30) and 26 to 21 at 16384; 1000 of 16 33 to 30 (38 to 26) and 21 to 24, 45 to 29 (49 to 30)
// and 39 to 24; 256 of 256 27 to 29 (31 to 23) and 14 to 24, 35 to 29 (39 to 31) and 25 to 23.  Past the LDS, with counters
// in memory and one block all the same: 300000 pages 302 to 27 and 319 to 23, 10^6 903 to 28 and 1115 to 27.
static bool one_block(int64_t batch, int64_t columns, int64_t pages) {
  return pages <= kSmallPages && batch * ((columns + 63) / 64) <= kSmallRows;
}

static int blocks_for(int64_t n, int each, int most) {
  const int64_t blocks = (n + each - 1) / each;
  return (int)(blocks < 1 ? 1 : blocks < most ? blocks : most);
}

static int entry_blocks(const PagesArgs& a) {
  return blocks_for((int64_t)((a.batch + kAhead - 1) / kAhead) * ((a.columns + 63) / 64), 4, 1024);
}

static int scan_blocks(const PagesArgs& a) { return blocks_for(a.pages, kEach * kPageThreads, kScanBlocks); }

static int launch_large_fork(const PagesArgs& a, hipStream_t stream) {
  const dim3 entries(entry_blocks(a)), scan(scan_blocks(a)), few(256), many(kPageThreads);
  hipLaunchKernelGGL(cache_fork_begin_kernel, dim3(blocks_for(a.pages > a.batch ? a.pages : a.batch, 256, 1024)), few, 0,
                     stream, a);
  TT_CHECK(launch_status("cache_fork_begin_kernel"));
  hipLaunchKernelGGL(cache_fork_count_kernel, entries, few, 0, stream, a);
  TT_CHECK(launch_status("cache_fork_count_kernel"));
  hipLaunchKernelGGL(cache_fork_rows_kernel, dim3(1), many, 0, stream, a);
  TT_CHECK(launch_status("cache_fork_rows_kernel"));
  hipLaunchKernelGGL(cache_count_kernel, scan, many, 0, stream, a, (const int*)a.hold, false);
  TT_CHECK(launch_status("cache_count_kernel"));
  hipLaunchKernelGGL(cache_fork_list_kernel, scan, many, 0, stream, a);
  TT_CHECK(launch_status("cache_fork_list_kernel"));
  hipLaunchKernelGGL(cache_fork_table_kernel, entries, few, 0, stream, a);
  return launch_status("cache_fork_table_kernel");
}

static int launch_large_compact(const PagesArgs& a, hipStream_t stream) {
  const dim3 scan(scan_blocks(a)), few(256), many(kPageThreads);
  hipLaunchKernelGGL(cache_count_kernel, scan, many, 0, stream, a, a.uses, true);
  TT_CHECK(launch_status("cache_count_kernel"));
  hipLaunchKernelGGL(cache_compact_list_kernel, scan, many, 0, stream, a);
  TT_CHECK(launch_status("cache_compact_list_kernel"));
  hipLaunchKernelGGL(cache_compact_moves_kernel, dim3(blocks_for(a.pages / 2, 256, 1024)), few, 0, stream, a);
  TT_CHECK(launch_status("cache_compact_moves_kernel"));
  hipLaunchKernelGGL(cache_compact_table_kernel, dim3(entry_blocks(a)), few, 0, stream, a);
  return launch_status("cache_compact_table_kernel");
}

constexpr int kParts = 32;        // tensors of one launch
constexpr int kCopyLoads = 8;      // 16 bytes a lane each
constexpr int kCopyBytes = kCopyLoads * 1024;  // of a page that a wave copies in one go

struct CopyArgs {
  char* data[kParts];
  int64_t page[kParts], row[kParts];  // bytes from a page to the next, and of one of its `rows` rows
  int rows[kParts], chunks[kParts];   // chunks: of the tensors up to this one
  int width[kParts];                  // bytes that a lane moves at once
  const int *source, *target, *tokens, *copies;  // tokens, copies: nullptr for whole pages, `count` of them
  int parts, count, pages, page_size;
};

// `bytes` that are less than a chunk or not aligned to 16.
template <typename W>
__device__ __forceinline__ void copy_rest(char* to, const char* from, int bytes, int lane) {
  const int n = bytes / (int)sizeof(W);
  for (int i = lane; i < n; i += 64) reinterpret_cast<W*>(to)[i] = reinterpret_cast<const W*>(from)[i];
  const int at = n * (int)sizeof(W) + lane;  // what is less than a W
  if (at < bytes) to[at] = from[at];
}

// A wave takes chunks of (copy, tensor, 8 KiB) in turn, each in loads that are all in flight at once (a block per chunk of
// 16 KiB: 217 us instead of 172, and 319 instead of 188 with pages of 16 tokens, half of whose pieces are scales of 8
// bytes).  Bound by HBM: 800 pages of 64 tokens in 8 halves of layers, in 8 bits with their scales, 164 us, 5.1 TB/s read and
// written.
__global__ __launch_bounds__(256) void cache_copy_kernel(CopyArgs a) {
  const int lane = threadIdx.x & 63, waves = (int)gridDim.x * 4;
  const int chunks = a.chunks[a.parts - 1];
  const int64_t items = (int64_t)(a.copies != nullptr ? *a.copies : a.count) * chunks;
  for (int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); item < items;
       item += waves) {
    // (32 bits wherever they do: a division in 64 takes a hundred instructions)
    const int c = items < (1LL << 32) ? (int)((uint32_t)item / (uint32_t)chunks) : (int)(item / chunks);
    const int chunk = (int)(item - (int64_t)c * chunks);
    const int from = a.source[c], to = a.target[c];
    if ((uint32_t)from >= (uint32_t)a.pages || (uint32_t)to >= (uint32_t)a.pages || from == to) continue;
    int part = 0;
    while (chunk >= a.chunks[part]) ++part;
    const int64_t begin = (int64_t)(chunk - (part > 0 ? a.chunks[part - 1] : 0)) * kCopyBytes;
    // the rows that hold `tokens` tokens
    int rows = a.rows[part];
    if (a.tokens != nullptr) rows = (int)(((int64_t)a.tokens[c] * rows + a.page_size - 1) / a.page_size);
    const int64_t left = rows * a.row[part] - begin;
    if (left <= 0) continue;
    char* const dst = a.data[part] + to * a.page[part] + begin;
    const char* const src = a.data[part] + from * a.page[part] + begin;
    if (a.width[part] == 16 && left >= kCopyBytes) {
      u32x4 x[kCopyLoads];
#pragma unroll
      for (int j = 0; j < kCopyLoads; ++j) x[j] = reinterpret_cast<const u32x4*>(src)[j * 64 + lane];
#pragma unroll
      for (int j = 0; j < kCopyLoads; ++j) reinterpret_cast<u32x4*>(dst)[j * 64 + lane] = x[j];
      continue;
    }
    const int bytes = (int)min(left, (int64_t)kCopyBytes);
    if (a.width[part] == 16) copy_rest<u32x4>(dst, src, bytes, lane);
    else if (a.width[part] == 4) copy_rest<uint32_t>(dst, src, bytes, lane);
    else copy_rest<char>(dst, src, bytes, lane);
  }
}

static int check_parts(const char* what, const tt_cache_part* parts, int count, int pages) {
  TT_REQUIRE(count >= 0 && (count == 0 || parts != nullptr), "%s: %d tensors", what, count);
  for (int i = 0; i < count; ++i) {
    const tt_cache_part& p = parts[i];
    TT_REQUIRE(p.data != nullptr && p.rows > 0 && p.row > 0 && p.page >= 0 && p.row <= (1LL << 40) / p.rows &&
                   (pages == 1 || p.page >= p.row * p.rows),
               "%s: tensor %d has pages of %d rows of %lld bytes, %lld apart", what, i, p.rows, (long long)p.row,
               (long long)p.page);
  }
  return TT_OK;
}

// The same copies in every tensor; `most` of them at most.
static int launch_copies(const tt_cache_part* parts, int count, const int* source, const int* target, const int* tokens,
                         const int* copies, int most, int pages, int page_size, hipStream_t stream) {
  for (int first = 0; first < count; first += kParts) {
    CopyArgs a{};
    a.parts = count - first < kParts ? count - first : kParts;
    int64_t chunks = 0;
    for (int i = 0; i < a.parts; ++i) {
      const tt_cache_part& p = parts[first + i];
      a.data[i] = static_cast<char*>(p.data), a.page[i] = p.page, a.row[i] = p.row, a.rows[i] = p.rows;
      const uint64_t grain = (uint64_t)(uintptr_t)p.data | (pages > 1 ? (uint64_t)p.page : 0);
      a.width[i] = (grain & 15) == 0 ? 16 : (grain & 3) == 0 ? 4 : 1;
      chunks += (p.row * p.rows + kCopyBytes - 1) / kCopyBytes;
      TT_REQUIRE(chunks < (1LL << 31), "cache_copy: pages of more than %d chunks", (1 << 30));
      a.chunks[i] = (int)chunks;
    }
    a.source = source, a.target = target, a.tokens = tokens, a.copies = copies;
    a.count = most, a.pages = pages, a.page_size = page_size;
    const int64_t blocks = (most * chunks + 3) / 4, full = 64 * (int64_t)device_cus();
    hipLaunchKernelGGL(cache_copy_kernel, dim3((unsigned)(blocks < full ? blocks : full)), dim3(256), 0, stream, a);
    const int rc = launch_status("cache_copy_kernel");
    if (rc != TT_OK) return rc;
  }
  return TT_OK;
}

static int64_t pages_list(int64_t batch, int64_t columns, int64_t pages) {
  return batch * columns < pages ? batch * columns : pages;
}

static int64_t pages_workspace(int64_t batch, int64_t columns, int64_t pages) {
  const int64_t copies = batch > pages / 2 ? batch : pages / 2;  // of a fork, and of a compaction
  const int64_t sums = one_block(batch, columns, pages) ? 0 : 2 + kScanBlocks;
  return 4 * (4 * batch + 2 * pages + pages_list(batch, columns, pages) + 3 * copies + 1 + sums);
}

static int check_state(const char* what, int batch, int columns, int pages, int page_size) {
  TT_REQUIRE(batch >= 0 && columns > 0, "%s: a page table of %d rows and %d columns", what, batch, columns);
  TT_CHECK(check_pages(what, pages, page_size, columns));
  TT_REQUIRE((int64_t)batch * columns < (1LL << 30) && pages < (1 << 30), "%s: %d rows of %d pages, and a cache of %d", what,
             batch, columns, pages);
  return TT_OK;
}

template <class C>
static PagesArgs pages_args(const C& c) {
  PagesArgs a{};
  a.table = c.table, a.lengths = c.lengths, a.uses = c.uses, a.new_table = c.new_table, a.new_uses = c.new_uses;
  a.table_row = c.table_row, a.batch = c.batch, a.columns = c.columns, a.pages = c.pages;
  a.page_shift = __builtin_ctz(c.page_size);
  a.list = (int)pages_list(c.batch, c.columns, c.pages);
  const int64_t copies = c.batch > c.pages / 2 ? c.batch : c.pages / 2;
  int* at = static_cast<int*>(c.workspace);
  const auto take = [&](int64_t n) {
    int* const p = at;
    at += n;
    return p;
  };
  a.rows = reinterpret_cast<int4*>(take(4 * (int64_t)c.batch));
  a.hold = take(c.pages), a.first = take(c.pages), a.free_pages = take(a.list);
  a.source = take(copies), a.target = take(copies), a.tokens = take(copies), a.copies = take(1);
  if (!one_block(c.batch, c.columns, c.pages)) a.needed = take(1), a.open = take(1), a.sums = take(kScanBlocks);
  return a;
}

}  // namespace tt

extern "C" int tt_cache_pages_workspace_bytes(int batch, int columns, int pages, int64_t* bytes) {
  using namespace tt;
  TT_CHECK(check_state("cache_pages", batch, columns, pages, 16));
  TT_REQUIRE(bytes != nullptr, "cache_pages: null pointer");
  *bytes = pages_workspace(batch, columns, pages);
  return TT_OK;
}

extern "C" int tt_cache_fork(const tt_cache_fork_pages* args, void* stream) {
  using namespace tt;
  TT_ARGS(tt_cache_fork_pages, "cache_fork");
  TT_CHECK(check_state("cache_fork", c.batch, c.columns, c.pages, c.page_size));
  TT_CHECK(check_parts("cache_fork", c.parts, c.part_count, c.pages));
  TT_REQUIRE(c.uses && c.new_uses && c.workspace && ((uintptr_t)c.workspace & 15) == 0 &&
                 c.workspace_bytes >= pages_workspace(c.batch, c.columns, c.pages),
             "cache_fork: null pointer, or a workspace of %lld bytes", (long long)c.workspace_bytes);
  TT_REQUIRE(c.batch == 0 || (c.table && c.lengths && c.new_table && c.new_lengths && c.table_row >= 0),
             "cache_fork: null pointer, or table_row %lld", (long long)c.table_row);
  PagesArgs a = pages_args(c);
  a.parents = c.parents, a.counts = c.counts, a.new_lengths = c.new_lengths;
  static std::atomic<uint64_t> ready{0};  // devices whose limit of dynamic LDS is raised
  if (one_block(c.batch, c.columns, c.pages))
    TT_CHECK(launch_pages("cache_fork_kernel", cache_fork_kernel, 16 * c.batch + 8 * c.pages, a, ready, (hipStream_t)stream));
  else
    TT_CHECK(launch_large_fork(a, (hipStream_t)stream));
  if (c.batch == 0) return TT_OK;
  return launch_copies(c.parts, c.part_count, a.source, a.target, a.tokens, a.copies, c.batch, c.pages, c.page_size,
                       (hipStream_t)stream);
}

extern "C" int tt_cache_compact(const tt_cache_compact_pages* args, void* stream) {
  using namespace tt;
  TT_ARGS(tt_cache_compact_pages, "cache_compact");
  TT_CHECK(check_state("cache_compact", c.batch, c.columns, c.pages, c.page_size));
  TT_CHECK(check_parts("cache_compact", c.parts, c.part_count, c.pages));
  TT_REQUIRE(c.uses && c.new_uses && c.workspace && ((uintptr_t)c.workspace & 15) == 0 &&
                 c.workspace_bytes >= pages_workspace(c.batch, c.columns, c.pages),
             "cache_compact: null pointer, or a workspace of %lld bytes", (long long)c.workspace_bytes);
  TT_REQUIRE(c.batch == 0 || (c.table && c.lengths && c.new_table && c.table_row >= 0),
             "cache_compact: null pointer, or table_row %lld", (long long)c.table_row);
  const PagesArgs a = pages_args(c);
  static std::atomic<uint64_t> ready{0};
  if (one_block(c.batch, c.columns, c.pages))
    TT_CHECK(launch_pages("cache_compact_kernel", cache_compact_kernel, 8 * c.pages, a, ready, (hipStream_t)stream));
  else
    TT_CHECK(launch_large_compact(a, (hipStream_t)stream));
  if (c.pages < 2) return TT_OK;
  return launch_copies(c.parts, c.part_count, a.source, a.target, nullptr, a.copies, c.pages / 2, c.pages, c.page_size,
                       (hipStream_t)stream);
}

extern "C" int tt_cache_copy(const tt_cache_copy_pages* args, void* stream) {
  using namespace tt;
  TT_ARGS(tt_cache_copy_pages, "cache_copy");
  TT_REQUIRE(c.count >= 0 && c.pages > 0, "cache_copy: %d copies in a cache of %d pages", c.count, c.pages);
  TT_CHECK(check_parts("cache_copy", c.parts, c.part_count, c.pages));
  if (c.count == 0) return TT_OK;
  TT_REQUIRE(c.source && c.target, "cache_copy: null pointer");
  return launch_copies(c.parts, c.part_count, c.source, c.target, nullptr, nullptr, c.count, c.pages, 1, (hipStream_t)stream);
}
