// Pages of a cache on the device: sequences forked, freed and extended by pages, pages moved to the cache's low end, and
// the copies of pages that both ask for.
//
// The state is a page table [batch, columns], lengths [batch] and uses [pages] (how many rows hold a page, and what holds
// the program has on it otherwise; 0: free).  One block works the new state out, phase by phase; a second launch copies.
#include "cache_checks.hpp"
#include "kernels.hpp"
#include "seq_attention.hpp"

namespace tt {

constexpr int kPageThreads = 1024;

// Counters that atomics of this launch change are read past the L1 (which may hold them as they were).
__device__ __forceinline__ int fresh(const int* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void put(int* p, int v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sum over the block's threads before this one; `total` over all.  (s_sums: an int per wave; free again at return.)
__device__ __forceinline__ int block_scan(int v, int* s_sums, int& total) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int upto = wave_scan_int(v);
  if (lane == 63) s_sums[wave] = upto;
  __syncthreads();
  const int sums = wave_scan_int(lane < kPageThreads / 64 ? s_sums[lane] : 0);
  total = __builtin_amdgcn_readlane(sums, kPageThreads / 64 - 1);
  const int before = wave > 0 ? __builtin_amdgcn_readlane(sums, max(wave - 1, 0)) : 0;
  __syncthreads();
  return before + upto - v;
}

struct PagesArgs {
  const int32_t *table, *lengths, *uses, *parents, *counts;
  int32_t *new_table, *new_lengths, *new_uses;
  int64_t table_row;
  int batch, columns, pages, page_shift, list;  // list: free pages that can be needed
  int *hold, *first, *free_pages;               // [pages], [pages], [list]
  int *begin, *whole;                           // [batch]
  int *source, *target, *tokens, *copies;       // copies to make, and their number
};

// What becomes of row b: the row that it continues (or -1), its length, and the tokens that it takes over.
struct ForkRow {
  int parent, after, kept;
};

__device__ __forceinline__ int held_pages(int tokens, int shift) { return (int)(((int64_t)tokens + (1 << shift) - 1) >> shift); }

__device__ __forceinline__ ForkRow fork_row(const PagesArgs& a, int b) {
  ForkRow r{-1, 0, 0};
  const int p = a.parents == nullptr ? b : a.parents[b];
  if ((uint32_t)p >= (uint32_t)a.batch) return r;
  const int most = a.columns << a.page_shift, before = min(max(a.lengths[p], 0), most);
  r.parent = p;
  r.after = (int)min(max((int64_t)before + (a.counts == nullptr ? 0 : a.counts[b]), (int64_t)0), (int64_t)most);
  r.kept = min(before, r.after);
  return r;
}

// Whole pages that a row takes over are shared.  One that it takes over in part is going to be written: of the rows that
// do so the first keeps it, if no row holds it whole and the program has no hold on it; the others get copies.  New pages
// are the lowest free ones, in the order of the rows.
__global__ __launch_bounds__(kPageThreads) void cache_fork_kernel(PagesArgs a) {
  __shared__ int s_sums[kPageThreads / 64];
  const int tid = threadIdx.x, entries = a.batch * a.columns, page = 1 << a.page_shift;
  for (int p = tid; p < a.pages; p += kPageThreads) {
    put(a.hold + p, a.uses[p]);
    put(a.first + p, a.batch);
  }
  __threadfence();
  __syncthreads();
  // Holds after the call: without the rows as they were, with the pages that rows keep whole.
  for (int e = tid; e < entries; e += kPageThreads) {
    const int b = e / a.columns, i = e - b * a.columns;
    const int length = min(max(a.lengths[b], 0), a.columns << a.page_shift);
    if (i < held_pages(length, a.page_shift)) {
      const int p = a.table[b * a.table_row + i];
      if ((uint32_t)p < (uint32_t)a.pages) atomicAdd(a.hold + p, -1);
    }
    const ForkRow r = fork_row(a, b);
    const int from = i << a.page_shift;
    if (from < r.kept) {
      const int p = a.table[r.parent * a.table_row + i];
      if ((uint32_t)p < (uint32_t)a.pages) {
        if (from + page <= r.kept) atomicAdd(a.hold + p, 1);
        else atomicMin(a.first + p, b);
      }
    }
  }
  __threadfence();
  __syncthreads();
  int needed = 0, copies = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kPageThreads) {
    const int b = b0 + tid;
    int need = 0, whole = 0, p = -1;
    ForkRow r{-1, 0, 0};
    bool copy = false;
    if (b < a.batch) {
      r = fork_row(a, b);
      whole = held_pages(r.kept, a.page_shift);
      if (r.kept & (page - 1)) {
        p = a.table[r.parent * a.table_row + whole - 1];
        if ((uint32_t)p < (uint32_t)a.pages) {
          // (only the first row of a page may find it unheld, and it alone changes that)
          if (fresh(a.first + p) == b && fresh(a.hold + p) == 0) put(a.hold + p, 1);
          else copy = true;
        }
      }
      whole -= copy ? 1 : 0;
      need = held_pages(r.after, a.page_shift) - whole;
    }
    int total;
    const int before = block_scan(need, s_sums, total);
    int copied;
    const int at = copies + block_scan(copy ? 1 : 0, s_sums, copied);
    if (b < a.batch) {
      put(a.begin + b, needed + before);
      put(a.whole + b, whole);
      a.new_lengths[b] = r.after;
      if (copy) {
        put(a.source + at, p);
        put(a.target + at, needed + before);  // its rank among the new pages so far
        put(a.tokens + at, r.kept & (page - 1));
      }
    }
    needed += total;
    copies += copied;
  }
  __threadfence();
  __syncthreads();
  int found = 0;
  for (int p0 = 0; p0 < a.pages; p0 += kPageThreads) {
    const int p = p0 + tid;
    const int hold = p < a.pages ? fresh(a.hold + p) : 1;
    if (p < a.pages) put(a.new_uses + p, hold);
    int total;
    const int rank = found + block_scan(hold == 0 ? 1 : 0, s_sums, total);
    if (hold == 0 && rank < min(needed, a.list)) put(a.free_pages + rank, p);
    found += total;
  }
  found = min(found, a.list);
  __threadfence();
  __syncthreads();
  for (int e = tid; e < entries; e += kPageThreads) {
    const int b = e / a.columns, i = e - b * a.columns;
    const ForkRow r = fork_row(a, b);
    const int whole = fresh(a.whole + b);
    int p = -1;
    if (i < whole) {
      p = a.table[r.parent * a.table_row + i];
    } else if (i < held_pages(r.after, a.page_shift)) {
      const int rank = fresh(a.begin + b) + i - whole;
      if (rank < found) {
        p = fresh(a.free_pages + rank);
        put(a.new_uses + p, 1);
      }
    }
    a.new_table[e] = p;
  }
  for (int c = tid; c < copies; c += kPageThreads) {
    const int rank = fresh(a.target + c);
    put(a.target + c, rank < found ? fresh(a.free_pages + rank) : -1);
  }
  if (tid == 0) *a.copies = copies;
}

// The used pages numbered from their count on move to the free ones below it, both in order: the fewest moves, none of
// which reads what another writes.
__global__ __launch_bounds__(kPageThreads) void cache_compact_kernel(PagesArgs a) {
  __shared__ int s_sums[kPageThreads / 64];
  const int tid = threadIdx.x, entries = a.batch * a.columns;
  int used = 0;
  for (int p = tid; p < a.pages; p += kPageThreads) used += a.uses[p] > 0 ? 1 : 0;
  int total;
  block_scan(used, s_sums, total);
  used = total;
  int from = 0, to = 0;
  for (int p0 = 0; p0 < a.pages; p0 += kPageThreads) {
    const int p = p0 + tid;
    const bool is_used = p < a.pages && a.uses[p] > 0;
    const bool moves = is_used && p >= used, fills = p < used && !is_used;
    const int r = from + block_scan(moves ? 1 : 0, s_sums, total);
    from += total;
    const int s = to + block_scan(fills ? 1 : 0, s_sums, total);
    to += total;
    if (moves) put(a.source + r, p);
    if (fills) put(a.target + s, p);
    if (p < a.pages) {
      put(a.new_uses + p, is_used && !moves ? a.uses[p] : 0);
      put(a.first + p, p);
    }
  }
  __threadfence();
  __syncthreads();
  for (int r = tid; r < from; r += kPageThreads) {
    const int p = fresh(a.source + r), q = fresh(a.target + r);
    put(a.first + p, q);
    put(a.new_uses + q, a.uses[p]);
  }
  __threadfence();
  __syncthreads();
  for (int e = tid; e < entries; e += kPageThreads) {
    const int b = e / a.columns, i = e - b * a.columns;
    const int length = min(max(a.lengths[b], 0), a.columns << a.page_shift);
    int p = -1;
    if (i < held_pages(length, a.page_shift)) {
      p = a.table[b * a.table_row + i];
      if ((uint32_t)p < (uint32_t)a.pages) p = fresh(a.first + p);
    }
    a.new_table[e] = p;
  }
  if (tid == 0) *a.copies = from;
}

constexpr int kParts = 32;        // tensors of one launch
constexpr int kCopyBytes = 16384;  // of a page that a block copies in one go

struct CopyArgs {
  char* data[kParts];
  int64_t page[kParts], row[kParts];  // bytes from a page to the next, and of one of its `rows` rows
  int rows[kParts], chunks[kParts];   // chunks: of the tensors up to this one
  int width[kParts];                  // bytes that a lane moves at once
  const int *source, *target, *tokens, *copies;  // tokens, copies: nullptr for whole pages, `count` of them
  int parts, count, pages, page_size;
};

template <typename W>
__device__ __forceinline__ void copy_run(char* to, const char* from, int bytes) {
  constexpr int N = kCopyBytes / 256 / 16;  // loads in flight
  const int n = bytes / (int)sizeof(W);
  for (int i0 = 0; i0 < n; i0 += 256 * N) {
    W x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = i0 + j * 256 + (int)threadIdx.x;
      if (i < n) x[j] = reinterpret_cast<const W*>(from)[i];
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = i0 + j * 256 + (int)threadIdx.x;
      if (i < n) reinterpret_cast<W*>(to)[i] = x[j];
    }
  }
  const int at = n * (int)sizeof(W) + (int)threadIdx.x;  // what is less than a W
  if (at < bytes) to[at] = from[at];
}

// A block takes chunks of (copy, tensor, 16 KiB) in turn.  Bound by HBM.
__global__ __launch_bounds__(256) void cache_copy_kernel(CopyArgs a) {
  const int chunks = a.chunks[a.parts - 1];
  const int64_t items = (int64_t)(a.copies != nullptr ? *a.copies : a.count) * chunks;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int c = (int)(item / chunks), chunk = (int)(item - (int64_t)c * chunks);
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
    const int bytes = (int)min(left, (int64_t)kCopyBytes);
    char* const dst = a.data[part] + to * a.page[part] + begin;
    const char* const src = a.data[part] + from * a.page[part] + begin;
    if (a.width[part] == 16) copy_run<u32x4>(dst, src, bytes);
    else if (a.width[part] == 4) copy_run<uint32_t>(dst, src, bytes);
    else copy_run<char>(dst, src, bytes);
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
    const int64_t items = most * chunks, full = 8 * (int64_t)device_cus();
    hipLaunchKernelGGL(cache_copy_kernel, dim3((unsigned)(items < full ? items : full)), dim3(256), 0, stream, a);
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
  return 4 * (2 * pages + pages_list(batch, columns, pages) + 2 * batch + 3 * copies + 1);
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
  a.hold = take(c.pages), a.first = take(c.pages), a.free_pages = take(a.list);
  a.begin = take(c.batch), a.whole = take(c.batch);
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
  TT_REQUIRE(c.uses && c.new_uses && c.workspace && ((uintptr_t)c.workspace & 3) == 0 &&
                 c.workspace_bytes >= pages_workspace(c.batch, c.columns, c.pages),
             "cache_fork: null pointer, or a workspace of %lld bytes", (long long)c.workspace_bytes);
  TT_REQUIRE(c.batch == 0 || (c.table && c.lengths && c.new_table && c.new_lengths && c.table_row >= 0),
             "cache_fork: null pointer, or table_row %lld", (long long)c.table_row);
  PagesArgs a = pages_args(c);
  a.parents = c.parents, a.counts = c.counts, a.new_lengths = c.new_lengths;
  hipLaunchKernelGGL(cache_fork_kernel, dim3(1), dim3(kPageThreads), 0, (hipStream_t)stream, a);
  TT_CHECK(launch_status("cache_fork_kernel"));
  if (c.batch == 0) return TT_OK;
  return launch_copies(c.parts, c.part_count, a.source, a.target, a.tokens, a.copies, c.batch, c.pages, c.page_size,
                       (hipStream_t)stream);
}

extern "C" int tt_cache_compact(const tt_cache_compact_pages* args, void* stream) {
  using namespace tt;
  TT_ARGS(tt_cache_compact_pages, "cache_compact");
  TT_CHECK(check_state("cache_compact", c.batch, c.columns, c.pages, c.page_size));
  TT_CHECK(check_parts("cache_compact", c.parts, c.part_count, c.pages));
  TT_REQUIRE(c.uses && c.new_uses && c.workspace && ((uintptr_t)c.workspace & 3) == 0 &&
                 c.workspace_bytes >= pages_workspace(c.batch, c.columns, c.pages),
             "cache_compact: null pointer, or a workspace of %lld bytes", (long long)c.workspace_bytes);
  TT_REQUIRE(c.batch == 0 || (c.table && c.lengths && c.new_table && c.table_row >= 0),
             "cache_compact: null pointer, or table_row %lld", (long long)c.table_row);
  const PagesArgs a = pages_args(c);
  hipLaunchKernelGGL(cache_compact_kernel, dim3(1), dim3(kPageThreads), 0, (hipStream_t)stream, a);
  TT_CHECK(launch_status("cache_compact_kernel"));
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
