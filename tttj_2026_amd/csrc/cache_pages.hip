// Pages of a cache on the device: sequences forked, freed and extended by pages, pages moved to the cache's low end, and
// the copies of pages that both ask for.
//
// The state is a page table [batch, columns], lengths [batch] and uses [pages] (how many rows hold a page, and what holds
// the program has on it otherwise; 0: free).  One block works the new state out, phase by phase; a second launch copies.
#include "cache_checks.hpp"
#include "kernels.hpp"
#include "seq_attention.hpp"

#include <atomic>

namespace tt {

constexpr int kPageThreads = 1024;
constexpr int kPageWaves = kPageThreads / 64;
constexpr int kEach = 4;              // pages that a thread looks at in turn
constexpr int kSmallPages = 16384;    // up to this many, counters lie in LDS (8 bytes a page) ...
constexpr int kSmallRows = 1024;      // ... and so do up to this many rows (16 bytes a row)

// Counters of the pages: in LDS, or for large caches in the workspace, where atomics change them and they are read past
// the L1 (which may hold them as they were).
template <bool SMALL>
struct Counters {
  int* at;
  __device__ __forceinline__ int get(int i) const {
    if constexpr (SMALL) return at[i];
    else return __hip_atomic_load(at + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __device__ __forceinline__ void put(int i, int v) const {
    if constexpr (SMALL) at[i] = v;
    else __hip_atomic_store(at + i, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __device__ __forceinline__ void add(int i, int v) const { atomicAdd(at + i, v); }
  __device__ __forceinline__ void least(int i, int v) const { atomicMin(at + i, v); }
};

template <bool SMALL>
__device__ __forceinline__ void phase() {  // what was written is read by others from here on
  if constexpr (!SMALL) __threadfence();
  __syncthreads();
}

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
//
// One block: each phase needs all that the one before it counted, and a barrier costs less than a launch.  A wave takes a
// row at a time, a lane a column.  Bound by latency: 4.7 us for 4 rows of 35 columns and 90 pages, 9.4 for 128 of 35 and 1493
// (33 with the counters in memory and a thread per entry).
template <bool SMALL>
__global__ __launch_bounds__(kPageThreads) void cache_fork_kernel(PagesArgs a) {
  extern __shared__ __align__(16) int pages_lds[];
  __shared__ int s_sums[kPageWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int shift = a.page_shift, page = 1 << shift;
  int4* const rows = SMALL ? reinterpret_cast<int4*>(pages_lds) : a.rows;
  int* const lds_pages = pages_lds + 4 * a.batch;
  const Counters<SMALL> hold{SMALL ? lds_pages : a.hold}, first{SMALL ? lds_pages + a.pages : a.first};
  // (the first rows of the pages are done with before the free ones are listed)
  const Counters<SMALL> free_pages{SMALL ? lds_pages + a.pages : a.free_pages};
  for (int b = tid; b < a.batch; b += kPageThreads) rows[b] = fork_row(a, b);
  for (int p = tid; p < a.pages; p += kPageThreads) {
    hold.put(p, a.uses[p]);
    first.put(p, a.batch);
  }
  phase<SMALL>();
  // Holds after the call: without the rows as they were, with the pages that rows keep whole.
  constexpr int AHEAD = 4;  // rows whose entries are asked for at once
  for (int b0 = wave; b0 < a.batch; b0 += AHEAD * kPageWaves)
    for (int i = lane; i < a.columns; i += 64) {
      int had[AHEAD], has[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        had[j] = has[j] = -1;
        const int b = b0 + j * kPageWaves;
        if (b >= a.batch) continue;
        const int4 r = rows[b];
        if (i < r.w) had[j] = a.table[b * a.table_row + i];
        if (i << shift < r.z) has[j] = a.table[r.x * a.table_row + i];
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        if ((uint32_t)had[j] < (uint32_t)a.pages) hold.add(had[j], -1);
        if ((uint32_t)has[j] < (uint32_t)a.pages) {
          const int b = b0 + j * kPageWaves;
          if ((i << shift) + page <= rows[b].z) hold.add(has[j], 1);
          else first.least(has[j], b);
        }
      }
    }
  phase<SMALL>();
  int needed = 0, copies = 0;
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
          if (first.get(p) == b && hold.get(p) == 0) hold.put(p, 1);
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
  phase<SMALL>();
  int found = 0;
  for (int p0 = 0; p0 < a.pages; p0 += kEach * kPageThreads) {
    int held[kEach], open = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int p = p0 + kEach * tid + j;
      held[j] = p < a.pages ? hold.get(p) : 1;
      open += held[j] == 0 ? 1 : 0;
    }
    int total, rank = block_scan(open, s_sums, total) + found;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int p = p0 + kEach * tid + j;
      if (p >= a.pages) continue;
      int uses = held[j];
      if (uses == 0) {
        if (rank < min(needed, a.list)) {
          free_pages.put(rank, p);
          uses = 1;
        }
        ++rank;
      }
      a.new_uses[p] = uses;
    }
    found += total;
  }
  found = min(found, min(needed, a.list));
  phase<SMALL>();
  for (int b0 = wave; b0 < a.batch; b0 += AHEAD * kPageWaves)
    for (int i = lane; i < a.columns; i += 64) {
      int p[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        p[j] = -1;
        const int b = b0 + j * kPageWaves;
        if (b >= a.batch) continue;
        const int4 r = rows[b];
        if (i < r.z) {
          p[j] = a.table[r.x * a.table_row + i];
        } else if (i < held_pages(r.y, shift)) {
          const int rank = r.w + i - r.z;
          if (rank < found) p[j] = free_pages.get(rank);
        }
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int b = b0 + j * kPageWaves;
        if (b < a.batch) a.new_table[(int64_t)b * a.columns + i] = p[j];
      }
    }
  for (int c = tid; c < copies; c += kPageThreads) {  // (a barrier and more since they were written)
    const int rank = rows[-1 - __hip_atomic_load(a.target + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)].w;
    a.target[c] = rank < found ? free_pages.get(rank) : -1;
  }
  if (tid == 0) *a.copies = copies;
}

// The used pages numbered from their count on move to the free ones below it, both in order: the fewest moves, none of
// which reads what another writes.
template <bool SMALL>
__global__ __launch_bounds__(kPageThreads) void cache_compact_kernel(PagesArgs a) {
  extern __shared__ __align__(16) int pages_lds[];
  __shared__ int s_sums[kPageWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // The number that a page gets; and the pages that move, then where to.
  const Counters<SMALL> number{SMALL ? pages_lds : a.first}, movers{SMALL ? pages_lds + a.pages : a.source};
  const Counters<SMALL> holes{SMALL ? pages_lds + a.pages + a.pages / 2 : a.target};
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
      if (moves) movers.put(r++, p);
      else if (p < used && uses[j] == 0) holes.put(s++, p);
      number.put(p, p);
      if (moves || p >= used) a.new_uses[p] = 0;
      else if (uses[j] > 0) a.new_uses[p] = uses[j];
    }
  }
  phase<SMALL>();
  for (int r = tid; r < moving; r += kPageThreads) {
    const int p = movers.get(r), q = holes.get(r);
    number.put(p, q);
    a.new_uses[q] = a.uses[p];
    if constexpr (SMALL) {
      a.source[r] = p;
      a.target[r] = q;
    }
  }
  phase<SMALL>();
  for (int b = wave; b < a.batch; b += kPageWaves) {
    const int held = held_pages(row_length(a, b), a.page_shift);
    for (int i = lane; i < a.columns; i += 64) {
      int p = -1;
      if (i < held) {
        p = a.table[b * a.table_row + i];
        if ((uint32_t)p < (uint32_t)a.pages) p = number.get(p);
      }
      a.new_table[(int64_t)b * a.columns + i] = p;
    }
  }
  if (tid == 0) *a.copies = moving;
}

// One block, with `lds` bytes where that is enough for the counters.
template <class K>
static int launch_pages(const char* what, K small, K large, bool fits, int lds, const PagesArgs& a, std::atomic<uint64_t>& ready,
                        hipStream_t stream) {
  if (fits) {
    int dev = 0;
    TT_HIP(hipGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if ((ready.load(std::memory_order_relaxed) & bit) == 0) {
      TT_HIP(hipFuncSetAttribute((const void*)small, hipFuncAttributeMaxDynamicSharedMemorySize,
                                 16 * kSmallRows + 8 * kSmallPages));
      ready.fetch_or(bit, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(small, dim3(1), dim3(kPageThreads), lds, stream, a);
  } else {
    hipLaunchKernelGGL(large, dim3(1), dim3(kPageThreads), 0, stream, a);
  }
  return launch_status(what);
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
  return 4 * (4 * batch + 2 * pages + pages_list(batch, columns, pages) + 3 * copies + 1);
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
  TT_CHECK(launch_pages("cache_fork_kernel", cache_fork_kernel<true>, cache_fork_kernel<false>,
                        c.pages <= kSmallPages && c.batch <= kSmallRows, 16 * c.batch + 8 * c.pages, a, ready,
                        (hipStream_t)stream));
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
  TT_CHECK(launch_pages("cache_compact_kernel", cache_compact_kernel<true>, cache_compact_kernel<false>,
                        c.pages <= kSmallPages, 8 * c.pages, a, ready, (hipStream_t)stream));
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
