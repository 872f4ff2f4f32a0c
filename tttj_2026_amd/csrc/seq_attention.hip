// Launches of the attention of ragged token rows (seq_attention.hpp): whole prompts, and new tokens over a paged
// cache; the merge of key ranges; the write of new keys and values into the cache.
#include "seq_attention.hpp"
#include "seq_launch.hpp"

namespace tt {

// The parts that a tile's keys were split into: `parts` of them, part p written by block first + p to its second entry
// where the tile's keys begin there, and to its first otherwise.
struct SeqParts {
  int first, parts;
};

__device__ __forceinline__ SeqParts seq_parts(const SeqShare& sh, int tile) {
  const int begin = sh.base + tile * sh.units.units;
  const int first = (begin + kSeqTileCost) / sh.share;
  return SeqParts{first, (begin + sh.units.units - 1) / sh.share - first + 1};
}

__device__ __forceinline__ int64_t seq_entry(const SeqAttnArgs& a, const SeqParts& t, int p, int hkv) {
  return (2 * (int64_t)(t.first + p) + (p == 0 ? 1 : 0)) * a.kv_heads + hkv;
}

// out = sum_s w_s O_s / sum_s w_s l_s over the shares s that a row's keys lie in, w_s = 2^(m_s - max m).  W waves per
// (token, head): head_dim / 4 lanes (rounded up to a power of two) take a part, the parts are dealt to 64 W / that
// many groups of lanes, four loads of each in flight, and the groups are added up at the end.  Rows of tiles that lie
// in one share were written by its block.  Bound by latency, that of five loads which depend on one another (first rows,
// lengths, sums, sums' weights): 5.9 us for 64 tokens on 32 heads of 128 (2 MiB read), 6.1 us for 4 tokens on
// 64 heads with 17 parts each (3 MiB).
template <typename T, int W>
__global__ __launch_bounds__(256) void seq_merge_kernel(SeqAttnArgs a, int rows_per_tile, int lanes) {
  __shared__ float s_sum[W > 1 ? W : 1][W > 1 ? 64 : 1][5];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = W > 1 ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave;
  if (row >= a.tokens * a.heads) return;
  const int token = row / a.heads, head = row - token * a.heads;
  int seq = token;
  if (a.starts != nullptr) {
    seq = seq_search(a.batch, token, [&](int b) { return seq_start(a.starts, b, a.tokens); });
    const int2 own = seq_rows(a, seq);
    if (token < own.x || token >= own.x + own.y) return;  // a row of no sequence
  }
  const SeqShare sh = seq_share(a, 0, seq, rows_per_tile);
  if (sh.total == 0) return;
  const SeqUnits u = sh.units;
  const int hkv = head / a.group;
  const int r = (token - u.first) * a.group + head - hkv * a.group;
  const int tile = r / rows_per_tile;
  const SeqParts t = seq_parts(sh, tile);
  const int parts = t.parts;
  if (parts == 1) return;
  const auto at = [&](int p) -> int64_t { return seq_entry(a, t, p, hkv) * rows_per_tile + r - tile * rows_per_tile; };
  float m = -INFINITY;
  for (int p = lane; p < parts; p += 64) m = fmaxf(m, a.part_ml[at(p)].x);
  for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
  const int in = lane & (lanes - 1), d = 4 * in;
  const int groups = 64 / lanes * W, group = (W > 1 ? wave * (64 / lanes) : 0) + lane / lanes;
  const bool live = d < a.head_dim;
  float l = 0.f;
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = group; p0 < parts; p0 += 4 * groups) {
    float2 y[4];
    floatx4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t e = at(min(p0 + i * groups, parts - 1));
      y[i] = a.part_ml[e];
      v[i] = *reinterpret_cast<const floatx4*>(a.part_o + e * a.head_dim + (live ? d : 0));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p0 + i * groups >= parts) break;
      // a part without a maximum saw no key (its sum, 0, is its weight) or only NaN (NaN is)
      const float w = y[i].x == -INFINITY ? y[i].y : seq_weight(y[i].x - m);
      l = fmaf(w, y[i].y, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(w, v[i][e], o[e]);
    }
  }
  for (int off = lanes; off < 64; off <<= 1) {
    l += __shfl_xor(l, off);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], off);
  }
  if constexpr (W > 1) {
    s_sum[wave][lane][4] = l;
#pragma unroll
    for (int e = 0; e < 4; ++e) s_sum[wave][lane][e] = o[e];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      l += s_sum[w][lane][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += s_sum[w][lane][e];
    }
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  typedef T v4 __attribute__((ext_vector_type(4)));
  if (live && lane < lanes)
    *reinterpret_cast<v4*>(static_cast<T*>(a.out) + (int64_t)row * a.head_dim + d) =
        v4{(T)(o[0] * inv), (T)(o[1] * inv), (T)(o[2] * inv), (T)(o[3] * inv)};
}

// The same for tiles of 128 rows, whose parts lie as wide_place says: W waves per 32 rows and 8 P features, each a
// W-th of the parts with a maximum and a sum of its own; lanes hold a row and 4 features of each 8.  Bound by latency as
// above where parts are few, then by reading them: 9.2 us for 3 chunks on heads of 256 (31 MiB, 3.2 TB/s).
template <typename T, int W, int P>
__global__ __launch_bounds__(64 * W) void seq_merge_wide_kernel(SeqAttnArgs a, int units) {
  __shared__ floatx4 s_o[W][P][64];
  __shared__ float2 s_ml[W][64];
  constexpr int R = 128;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int unit = (int)blockIdx.x % units, rest = (int)blockIdx.x / units;
  const int rw = rest & 3, hkv = (rest >> 2) % a.kv_heads;
  const SeqTile sq = seq_tile(a, (rest >> 2) / a.kv_heads, R);
  const int r = 32 * rw + (lane & 31), rows = sq.count * a.group - sq.tile * R;  // row of the tile; rows from there on
  if (sq.tile < 0 || 32 * rw >= rows) return;
  const SeqShare sh = seq_share(a, 0, sq.seq, R);
  if (sh.total == 0) return;
  const SeqParts t = seq_parts(sh, sq.tile);
  if (t.parts == 1) return;
  const int d0 = 8 * P * unit, hd = a.head_dim;
  const int place = wide_place(hd, r, d0 + 4 * (lane >> 5));
  float m = -INFINITY, l = 0.f;
  floatx4 o[P];
#pragma unroll
  for (int g = 0; g < P; ++g) o[g] = floatx4{0.f, 0.f, 0.f, 0.f};
  // A part (or a wave) without a maximum saw no key (its sum, 0, is its weight) or only NaN (NaN is).
  const auto weight = [&](float2 ml) -> float {
    return ml.x == -INFINITY ? ml.y : seq_weight(ml.x - m);
  };
  const bool own = r < rows;  // entries of rows behind the last are not written
  for (int p0 = wave; p0 < t.parts; p0 += 4 * W) {
    float2 y[4];
    floatx4 v[4][P];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t e = seq_entry(a, t, min(p0 + i * W, t.parts - 1), hkv) * R;
      y[i] = make_float2(-INFINITY, 0.f);
      if (own) y[i] = a.part_ml[e + r];
#pragma unroll
      for (int g = 0; g < P; ++g) {
        v[i][g] = floatx4{0.f, 0.f, 0.f, 0.f};
        if (own && d0 + 8 * g < hd) v[i][g] = *reinterpret_cast<const floatx4*>(a.part_o + e * hd + place + 256 * g);
      }
    }
    float m_new = m;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p0 + i * W < t.parts) m_new = fmaxf(m_new, y[i].x);
    const float corr = m_new == -INFINITY ? 1.f : seq_weight(m - m_new);
    m = m_new;
    l *= corr;
#pragma unroll
    for (int g = 0; g < P; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[g][e] *= corr;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p0 + i * W >= t.parts) break;
      const float w = weight(y[i]);
      l = fmaf(w, y[i].y, l);
#pragma unroll
      for (int g = 0; g < P; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[g][e] = fmaf(w, v[i][g][e], o[g][e]);
    }
  }
#pragma unroll
  for (int g = 0; g < P; ++g) s_o[wave][g][lane] = o[g];
  s_ml[wave][lane] = make_float2(m, l);
  __syncthreads();
  if (wave >= P || !own || d0 + 8 * wave >= hd) return;
  float2 y[W];
  m = -INFINITY;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    y[w] = s_ml[w][lane];
    m = fmaxf(m, y[w].x);
  }
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
  l = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const float f = weight(y[w]);
    const floatx4 x = s_o[w][wave][lane];
    l = fmaf(f, y[w].y, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = fmaf(f, x[e], sum[e]);
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const int row = sq.tile * R + r, token = row / a.group;
  typedef T v4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<v4*>(static_cast<T*>(a.out) +
                         ((int64_t)(sq.first + token) * a.heads + hkv * a.group + row - token * a.group) * hd + d0 +
                         8 * wave + 4 * (lane >> 5)) =
      v4{(T)(sum[0] * inv), (T)(sum[1] * inv), (T)(sum[2] * inv), (T)(sum[3] * inv)};
}

template <typename T>
static int launch_seq_merge_wide(const SeqAttnArgs& a, int tiles, bool many_parts, hipStream_t stream) {
  const int pieces = a.head_dim / 8, units = many_parts ? pieces : (pieces + 3) / 4;
  const int blocks = tiles * a.kv_heads * 4 * units;
  if (many_parts)
    hipLaunchKernelGGL((seq_merge_wide_kernel<T, 16, 1>), dim3(blocks), dim3(1024), 0, stream, a, units);
  else
    hipLaunchKernelGGL((seq_merge_wide_kernel<T, 4, 4>), dim3(blocks), dim3(256), 0, stream, a, units);
  return launch_status("seq_merge_wide_kernel");
}

template <typename T>
static int launch_seq_merge(const SeqAttnArgs& a, int rows_per_tile, bool many_parts, hipStream_t stream) {
  int lanes = 2;
  while (4 * lanes < a.head_dim) lanes *= 2;
  const int rows = a.tokens * a.heads;
  if (many_parts)  // a block per row, else a wave
    hipLaunchKernelGGL((seq_merge_kernel<T, 4>), dim3(rows), dim3(256), 0, stream, a, rows_per_tile, lanes);
  else
    hipLaunchKernelGGL((seq_merge_kernel<T, 1>), dim3(rows / 4 + 1), dim3(256), 0, stream, a, rows_per_tile, lanes);
  return launch_status("seq_merge_kernel");
}

struct AppendArgs {
  const uint16_t *k, *v;
  uint16_t *k_cache, *v_cache;
  const int32_t *starts, *lengths, *table;
  int64_t k_row, k_head, v_row, v_head, kc_page, kc_row, kc_head, vc_page, vc_row, vc_head, table_row;
  int tokens, batch, heads, chunks;  // per token: `heads` runs of `chunks` 16-byte pieces
  int pages, table_pages, page_shift;
};

// One wave per token: its K and V rows go to their place in the cache, 16 bytes a lane.  No computation: bound by HBM
// (36000 tokens on 8 heads of 128 45 us, 6.5 TB/s read and written, with part of it in the last level cache; 59 us a call
// in a stream of such calls), and by the call for few (64 tokens: 3.3 us of 8.2).
__global__ __launch_bounds__(256) void cache_append_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 63;
  const int token = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (token >= a.tokens) return;
  int seq = token, i = 0, count = 1;
  if (a.starts != nullptr) {
    seq = seq_search(a.batch, token, [&](int b) { return seq_start(a.starts, b, a.tokens); });
    const int first = seq_start(a.starts, seq, a.tokens);
    i = token - first;
    count = seq_start(a.starts, seq + 1, a.tokens) - first;
    if (i < 0 || i >= count) return;
  }
  const int64_t at = (int64_t)a.lengths[seq] - count + i;
  if (at < 0 || (at >> a.page_shift) >= a.table_pages) return;
  const int page = a.table[seq * a.table_row + (at >> a.page_shift)];
  if ((uint32_t)page >= (uint32_t)a.pages) return;
  const int in = (int)at & ((1 << a.page_shift) - 1);
  const uint16_t* k = a.k + token * a.k_row;
  const uint16_t* v = a.v + token * a.v_row;
  uint16_t* kc = a.k_cache + page * a.kc_page + in * a.kc_row;
  uint16_t* vc = a.v_cache + page * a.vc_page + in * a.vc_row;
  for (int c = lane; c < a.heads * a.chunks; c += 64) {
    const int h = a.heads == 1 ? 0 : c / a.chunks, e = (c - h * a.chunks) * 8;
    const u32x4 x = *reinterpret_cast<const u32x4*>(k + h * a.k_head + e);
    const u32x4 y = *reinterpret_cast<const u32x4*>(v + h * a.v_head + e);
    *reinterpret_cast<u32x4*>(kc + h * a.kc_head + e) = x;
    *reinterpret_cast<u32x4*>(vc + h * a.vc_head + e) = y;
  }
}

int launch_seq_attention(const SeqAttnArgs& a, bool paged, SeqShape shape, int dtype, hipStream_t stream) {
  if (a.head_dim > 128) return launch_seq_attention_wide(a, paged, shape, dtype, stream);
  if (a.head_dim > 64) return launch_seq_hd<128>(a, paged, shape, dtype, stream);
  if (a.head_dim > 32) return launch_seq_hd<64>(a, paged, shape, dtype, stream);
  return launch_seq_hd<32>(a, paged, shape, dtype, stream);
}

// Blocks of a kernel that a CU holds (its registers, and its LDS: 16, 32, 64 or 128 KiB and a little more each).
static int seq_resident(bool wide, int head_dim, int bytes) {
  if (wide) return head_dim <= 64 ? 3 : head_dim <= 128 ? 2 : 1;
  if (bytes > 1) return head_dim <= 64 && bytes == 2 ? 4 : 2;
  if (bytes) return head_dim <= 64 ? 4 : head_dim <= 128 ? 2 : 4;
  return head_dim <= 32 ? 6 : head_dim <= 64 ? 4 : 2;
}

// How a call is given to blocks.  Figures: MI355X, us per call, heads of 128 unless another width is named.
struct SeqPlan {
  SeqShape shape;
  int rows;  // of a block
  int tiles;  // per kv head, at most
  int slots, mode;
  int64_t part_rows;  // rows of the workspace
  bool many_parts;
};

// max_length < 0: packed sequences (no keys but their own).  bytes: over an 8-bit cache, the heads that share a narrow block.
static SeqPlan seq_plan(int64_t tokens, int batch, int heads, int kv_heads, int head_dim, int64_t held, int max_length,
                        bool single, int bytes = 0) {
  SeqPlan p{};
  const int64_t G = heads / kv_heads;
  const int cus = device_cus();
  const bool paged = max_length >= 0;
  // 128 rows share every tile of keys that they read, 32 rows waste fewer products on rows that are not there.  With
  // 40 / 64 / 96 rows a sequence, 16 sequences of 2000 keys on 4 heads: 32-row tiles 27.8 / 28.3 / 28.4, 128-row tiles
  // 27.9 / 29 / 32; but 64 rows over 4000 keys, 64 sequences on 8 heads: 377 and 191 (every key is read twice).
  const bool wide = !paged || (single ? G > 32 : tokens * G > 32 * (int64_t)batch);
  p.rows = wide ? 128 : 32;
  const int64_t tiles = single ? tokens * ((G + p.rows - 1) / p.rows) : tokens * G / p.rows + batch;
  const int64_t blocks = tiles * kv_heads, held_blocks = (int64_t)seq_resident(wide, head_dim, bytes) * cus;
  // Up to a block per CU the waves of a block are as many as its LDS feeds, else two: 16 sequences of 4 tokens, 1000 keys
  // on 4 heads of 64, 17.4 with two waves and 12.3 with eight; 16 drafts of 1 to 7 tokens, to 2100 keys, 28.3 and 14.8.
  p.shape = wide ? SeqShape::kWide : blocks <= cus ? SeqShape::kDeep : SeqShape::kNarrow;
  p.tiles = p.slots = (int)tiles;
  p.mode = kSeqInOrder;
  // Keys up to which a block takes a tile alone, in rounds of the block's waves: dealing keys out costs a second launch,
  // and parts that are written and read.  Measured on MI355X per call, alone -> in shares: 16 blocks of 8 waves on
  // heads of 64, 1000 keys (4 rounds) 9.3 -> 11.0 us, 2000 12.9 -> 11.5; 8 blocks of 4 on heads of 128, 500 keys 9.9 ->
  // 12.4, 1000 (8 rounds) 14.1 -> 12.7.  Blocks that fill a good part of the chip gain less: 256 on heads of 64, 4000
  // keys (16 rounds) 46 -> 50, 8000 99 -> 105; 128 on heads of 128, 2000 (16) 27 -> 30, 4000 49 -> 48, and with lengths
  // from 1 to 4000 39 -> 32; 512 of two waves on heads of 128, 1000 keys (16) 43 -> 47, lengths to 4000 125 -> 107; 512 of
  // one wave on heads of 256, 700 keys (22) 66 -> 69, lengths to 700 43.3 -> 42.5, to 1020 60 -> 54; 300 of one, 700 keys
  // 42 -> 49, lengths to 700 40 -> 34.
  const int keys_per_round = wide    ? 64
                             : bytes ? seq8_keys(head_dim) * (p.shape == SeqShape::kNarrow && bytes > 1
                                                                  ? 1
                                                                  : seq8_waves(p.shape, head_dim))
                                     : 32 * seq_waves(p.shape, head_dim);
  int rounds = blocks <= cus / 4 ? 6 : 16;
  // Over an 8-bit cache rounds are longer (64 keys a wave on heads to 128) and bytes fewer.  Alone -> in shares, uniform
  // lengths | from 1 on: 256 blocks on heads of 64, 1000 keys (2 rounds) 17.6 -> 18.8 | 13.5 -> 14.8, 2000 28.8 -> 23.8 | 22 ->
  // 20; 128, 2000 (4) 19.3 -> 19.2 | 16 -> 15, 16 drafts of 1 to 7 tokens to 2100 16.5 -> 18; 32 on heads of 128, 1000 keys
  // (4) 14.3 -> 17.4, 2000 21 -> 17.5; 128, 2000 (8) 24.5 -> 24.7 | 23 -> 21, 4000 38 -> 33; 16 on heads of 256, 1000 (8)
  // 22.6 -> 23.6, 2000 35 -> 22; 256, 2000 (16) 49 -> 52 | 38 -> 34; 512 narrow ones on heads of 64, 500 (8) 16.6 -> 18.2 |
  // 16 -> 15, 1000 28 -> 23; on heads of 128, 500 21 -> 25 | 20 -> 20, 1000 34 -> 35 | 34 -> 26; 1024 on heads of 64, 1000
  // (16) 30 -> 34 | 28 -> 25, 2000 53 -> 54 | 49 -> 34.
  if (bytes && !wide) {
    if (p.shape == SeqShape::kNarrow) rounds = head_dim <= 128 && blocks <= 2 * cus ? 10 : 16;
    else if (head_dim <= 64) rounds = blocks <= cus / 2 ? 5 : 3;
    else rounds = (head_dim <= 128 ? 5 : 8) * (blocks <= cus / 4 ? 1 : 2);
  }
  const int alone = rounds * keys_per_round;
  // Beyond the blocks that the chip holds (four times as many of 32 rows), tiles spread by themselves: 1088 tiles of 128
  // rows over 500 to 4600 keys, 195 alone and 272 in shares; 800 of 32 rows over 1 to 4000 keys, 193 and 162.
  // Heads that share a block count as one, for as many sequences as that pays: lengths from 1 to 2000 on 16 heads of 64, 128
  // sequences 61 -> 53; 256 to 1500 112 -> 94; but 512 of 1100 keys on 4 heads 52 -> 63.
  const int64_t most = (wide ? 1 : 4) * held_blocks, placed = !wide && bytes > 1 && batch <= 256 ? blocks / bytes : blocks;
  if (paged && max_length > alone && batch <= 512 && placed < most &&
      tiles * (held / kSeqUnit + 1 + kSeqTileCost) + held_blocks < (1LL << 31)) {
    p.mode = kSeqShares;
    if (!wide) p.shape = SeqShape::kNarrow;
    const int64_t units = tiles * ((max_length + kSeqUnit - 1) / kSeqUnit + kSeqTileCost);
    int64_t slots = held_blocks / (!wide && bytes > 1 ? kv_heads / bytes : kv_heads);
    if (slots > (units + kSeqMinShare - 1) / kSeqMinShare) slots = (units + kSeqMinShare - 1) / kSeqMinShare;
    p.slots = (int)(slots > 1 ? slots : 1);
    p.part_rows = 2 * (int64_t)p.slots * kv_heads * p.rows;
    // Many parts of few rows are joined by more waves each: one chunk of 16 tokens over 30000 keys on one head (8 query
    // heads) 29.4 -> 23.5, but 4 of them over 8000 keys on 8 heads (16 parts a tile) 35 -> 48; 4 single tokens over
    // 100000 keys 287 -> 284.5, but 64 over 1 to 4000 keys 106 -> 107.5.
    p.many_parts = p.slots > (wide ? 32 : 8) * tiles && tokens * heads <= 2048;
  } else if (!single && batch <= 64 && blocks > held_blocks && tokens * G < (1LL << 30)) {
    // More tiles than the chip holds: the last to start should be the shortest.  2 prompts of 4096 tokens on 16 heads of
    // 64 in order 106, heaviest first 91; 12 prompts of very different lengths 123 and 123.
    p.mode = kSeqHeaviest;
  }
  return p;
}

}  // namespace tt

extern "C" int tt_packed_attention_fwd(const tt_packed_attention* args, void* stream) {
  using namespace tt;
  TT_ARGS(tt_packed_attention, "packed_attention");
  TT_CHECK(check_heads("packed_attention", c.tokens, c.batch, c.heads, c.kv_heads, c.head_dim, c.dtype));
  TT_REQUIRE(c.scale > 0.f && c.scale < 2e38f, "packed_attention: scale %g is not positive and finite", c.scale);
  if (c.tokens == 0 || c.batch == 0) return TT_OK;
  TT_REQUIRE(c.q && c.k && c.v && c.starts && c.out, "packed_attention: null pointer");
  TT_CHECK(check_rows("packed_attention: q", c.q, c.q_row, c.q_head));
  TT_CHECK(check_rows("packed_attention: k", c.k, c.k_row, c.k_head));
  TT_CHECK(check_rows("packed_attention: v", c.v, c.v_row, c.v_head));
  TT_CHECK(check_rows("packed_attention: out", c.out, 0, 0));
  SeqAttnArgs a{};
  a.q = c.q, a.k = c.k, a.v = c.v, a.out = c.out, a.starts = c.starts;
  a.q_row = c.q_row, a.q_head = c.q_head, a.k_row = c.k_row, a.k_head = c.k_head, a.v_row = c.v_row, a.v_head = c.v_head;
  a.tokens = c.tokens, a.batch = c.batch, a.heads = c.heads, a.kv_heads = c.kv_heads, a.group = c.heads / c.kv_heads;
  a.head_dim = c.head_dim, a.causal = c.causal != 0, a.scale_log2 = c.scale * 1.4426950408889634f;
  const SeqPlan p = seq_plan(c.tokens, c.batch, c.heads, c.kv_heads, c.head_dim, 0, -1, false);
  a.slots = p.slots, a.mode = p.mode;
  return launch_seq_attention(a, false, SeqShape::kWide, c.dtype, (hipStream_t)stream);
}

namespace tt {

static int workspace_bytes(const char* what, bool bytes_cache, int tokens, int batch, int heads, int kv_heads, int head_dim,
                           int page_size, int table_pages, int max_length, int single, int64_t* bytes) {
  TT_CHECK(check_heads(what, tokens, batch, heads, kv_heads, head_dim, TT_FP16));
  if (bytes_cache) TT_CHECK(check_head8(what, head_dim));
  TT_CHECK(check_pages(what, 1, page_size, table_pages));
  TT_REQUIRE(max_length >= 0 && bytes != nullptr, "%s: max_length %d", what, max_length);
  *bytes = 0;
  if (tokens == 0 || batch == 0) return TT_OK;
  // (which heads lie side by side is not known here: the most that either needs)
  for (int side_by_side = 0; side_by_side < (bytes_cache ? 2 : 1); ++side_by_side) {
    const int shared = !bytes_cache ? 0 : side_by_side ? seq8_heads(head_dim, kv_heads, head_dim, head_dim) : 1;
    const int64_t need = 4 * (head_dim + 2) * seq_plan(tokens, batch, heads, kv_heads, head_dim,
                                                       (int64_t)page_size * table_pages, max_length, single != 0,
                                                       shared).part_rows;
    if (need > *bytes) *bytes = need;
  }
  return TT_OK;
}

// What both forms of the cache have in common: the checks of a call, and its launches.
template <class C>
static int check_cache_attention(const char* what, const C& c) {
  TT_CHECK(check_heads(what, c.tokens, c.batch, c.heads, c.kv_heads, c.head_dim, c.dtype));
  TT_CHECK(check_pages(what, c.pages, c.page_size, c.table_pages));
  TT_REQUIRE(c.scale > 0.f && c.scale < 2e38f, "%s: scale %g is not positive and finite", what, c.scale);
  TT_REQUIRE(c.max_length >= 0, "%s: max_length %d", what, c.max_length);
  if (c.tokens == 0 || c.batch == 0) return TT_OK;
  TT_REQUIRE(c.q && c.k_cache && c.v_cache && c.table && c.lengths && c.out, "%s: null pointer", what);
  TT_REQUIRE(c.starts != nullptr || c.tokens == c.batch, "%s: %d tokens for %d sequences without starts", what, c.tokens,
             c.batch);
  TT_CHECK(check_rows("cache_attention: q", c.q, c.q_row, c.q_head));
  TT_REQUIRE(c.k_page >= 0 && c.v_page >= 0 && c.table_row >= 0, "%s: page strides %lld, %lld", what, (long long)c.k_page,
             (long long)c.v_page);
  return check_rows("cache_attention: out", c.out, 0, 0);
}

template <class C>
static int run_cache_attention(const char* what, const C& c, SeqAttnArgs& a, bool bytes_cache, hipStream_t stream) {
  const SeqPlan p = seq_plan(c.tokens, c.batch, c.heads, c.kv_heads, c.head_dim, (int64_t)c.page_size * c.table_pages,
                             c.max_length, c.starts == nullptr,
                             bytes_cache ? seq8_heads(c.head_dim, c.kv_heads, c.k_head, c.v_head) : 0);
  const int64_t bytes = 4 * (c.head_dim + 2) * p.part_rows;
  TT_REQUIRE(bytes == 0 || (c.workspace != nullptr && c.workspace_bytes >= bytes && ((uintptr_t)c.workspace & 15) == 0),
             "%s: a workspace of %lld bytes is needed, %lld given", what, (long long)bytes, (long long)c.workspace_bytes);
  a.q = c.q, a.k = c.k_cache, a.v = c.v_cache, a.out = c.out, a.starts = c.starts, a.lengths = c.lengths, a.table = c.table;
  a.q_row = c.q_row, a.q_head = c.q_head, a.k_row = c.k_row, a.k_head = c.k_head, a.v_row = c.v_row, a.v_head = c.v_head;
  a.k_page = c.k_page, a.v_page = c.v_page, a.table_row = c.table_row;
  a.tokens = c.tokens, a.batch = c.batch, a.heads = c.heads, a.kv_heads = c.kv_heads, a.group = c.heads / c.kv_heads;
  a.head_dim = c.head_dim, a.pages = c.pages, a.table_pages = c.table_pages, a.page_shift = __builtin_ctz(c.page_size);
  a.causal = 1, a.scale_log2 = c.scale * 1.4426950408889634f;
  a.slots = p.slots, a.mode = p.mode;
  a.part_o = static_cast<float*>(c.workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + p.part_rows * c.head_dim);
  TT_CHECK(bytes_cache ? launch_seq8_attention(a, p.shape, c.dtype, stream)
                       : launch_seq_attention(a, true, p.shape, c.dtype, stream));
  if (p.mode != kSeqShares) return TT_OK;
  if (p.shape == SeqShape::kWide)
    return c.dtype == TT_FP16 ? launch_seq_merge_wide<half>(a, p.tiles, p.many_parts, stream)
                              : launch_seq_merge_wide<bf16>(a, p.tiles, p.many_parts, stream);
  return c.dtype == TT_FP16 ? launch_seq_merge<half>(a, p.rows, p.many_parts, stream)
                          : launch_seq_merge<bf16>(a, p.rows, p.many_parts, stream);
}

}  // namespace tt

extern "C" int tt_cache_attention_workspace_bytes(int tokens, int batch, int heads, int kv_heads, int head_dim,
                                                  int page_size, int table_pages, int max_length, int single,
                                                  int64_t* bytes) {
  return tt::workspace_bytes("cache_attention", false, tokens, batch, heads, kv_heads, head_dim, page_size, table_pages,
                             max_length, single, bytes);
}

extern "C" int tt_cache_attention8_workspace_bytes(int tokens, int batch, int heads, int kv_heads, int head_dim,
                                                   int page_size, int table_pages, int max_length, int single,
                                                   int64_t* bytes) {
  return tt::workspace_bytes("cache_attention", true, tokens, batch, heads, kv_heads, head_dim, page_size, table_pages,
                             max_length, single, bytes);
}

extern "C" int tt_cache_attention_fwd(const tt_cache_attention* args, void* stream) {
  using namespace tt;
  TT_ARGS(tt_cache_attention, "cache_attention");
  TT_CHECK(check_cache_attention("cache_attention", c));
  if (c.tokens == 0 || c.batch == 0) return TT_OK;
  TT_CHECK(check_rows("cache_attention: k_cache", c.k_cache, c.k_row, c.k_head));
  TT_CHECK(check_rows("cache_attention: v_cache", c.v_cache, c.v_row, c.v_head));
  TT_REQUIRE(c.k_page % 8 == 0 && c.v_page % 8 == 0, "cache_attention: page strides %lld, %lld", (long long)c.k_page,
             (long long)c.v_page);
  SeqAttnArgs a{};
  return run_cache_attention("cache_attention", c, a, false, (hipStream_t)stream);
}

extern "C" int tt_cache_attention8_fwd(const tt_cache_attention8* args, void* stream) {
  using namespace tt;
  TT_ARGS(tt_cache_attention8, "cache_attention");
  TT_CHECK(check_cache_attention("cache_attention", c));
  TT_CHECK(check_head8("cache_attention", c.head_dim));
  TT_CHECK(check_block("cache_attention", c.block, c.page_size));
  if (c.tokens == 0 || c.batch == 0) return TT_OK;
  TT_CHECK(check_rows8("cache_attention: k_cache", c.k_cache, c.k_page, c.k_row, c.k_head));
  TT_CHECK(check_rows8("cache_attention: v_cache", c.v_cache, c.v_page, c.v_row, c.v_head));
  TT_CHECK(check_scales("cache_attention", c));
  SeqAttnArgs a{};
  a.k_scale = c.k_scales, a.v_scale = c.v_scales, a.block_shift = __builtin_ctz(c.block);
  a.s_page = (int)c.s_page, a.s_block = (int)c.s_block, a.s_head = (int)c.s_head;
  return run_cache_attention("cache_attention", c, a, true, (hipStream_t)stream);
}

extern "C" int tt_cache_append(const tt_cache_rows* args, void* stream) {
  using namespace tt;
  TT_ARGS(tt_cache_rows, "cache_append");
  TT_CHECK(check_heads("cache_append", c.tokens, c.batch, c.kv_heads, c.kv_heads, c.head_dim, TT_FP16));
  TT_CHECK(check_pages("cache_append", c.pages, c.page_size, c.table_pages));
  TT_REQUIRE(c.tokens < (1 << 26), "cache_append: %d tokens are more than one launch takes", c.tokens);
  if (c.tokens == 0 || c.batch == 0) return TT_OK;
  TT_REQUIRE(c.k && c.v && c.k_cache && c.v_cache && c.table && c.lengths, "cache_append: null pointer");
  TT_REQUIRE(c.starts != nullptr || c.tokens == c.batch, "cache_append: %d tokens for %d sequences without starts",
             c.tokens, c.batch);
  TT_CHECK(check_rows("cache_append: k", c.k, c.k_row, c.k_head));
  TT_CHECK(check_rows("cache_append: v", c.v, c.v_row, c.v_head));
  TT_CHECK(check_rows("cache_append: k_cache", c.k_cache, c.kc_row, c.kc_head));
  TT_CHECK(check_rows("cache_append: v_cache", c.v_cache, c.vc_row, c.vc_head));
  TT_REQUIRE(c.kc_page % 8 == 0 && c.vc_page % 8 == 0 && c.kc_page >= 0 && c.vc_page >= 0 && c.table_row >= 0,
             "cache_append: page strides %lld, %lld", (long long)c.kc_page, (long long)c.vc_page);
  AppendArgs a{};
  a.k = static_cast<const uint16_t*>(c.k), a.v = static_cast<const uint16_t*>(c.v);
  a.k_cache = static_cast<uint16_t*>(c.k_cache), a.v_cache = static_cast<uint16_t*>(c.v_cache);
  a.starts = c.starts, a.lengths = c.lengths, a.table = c.table;
  a.k_row = c.k_row, a.k_head = c.k_head, a.v_row = c.v_row, a.v_head = c.v_head;
  a.kc_page = c.kc_page, a.kc_row = c.kc_row, a.kc_head = c.kc_head;
  a.vc_page = c.vc_page, a.vc_row = c.vc_row, a.vc_head = c.vc_head, a.table_row = c.table_row;
  a.tokens = c.tokens, a.batch = c.batch, a.heads = c.kv_heads, a.chunks = c.head_dim / 8;
  if (c.k_head == c.head_dim && c.v_head == c.head_dim && c.kc_head == c.head_dim && c.vc_head == c.head_dim)
    a.heads = 1, a.chunks = c.kv_heads * (c.head_dim / 8);  // the heads of a token lie side by side everywhere
  a.pages = c.pages, a.table_pages = c.table_pages, a.page_shift = __builtin_ctz(c.page_size);
  hipLaunchKernelGGL(cache_append_kernel, dim3((unsigned)((c.tokens + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a);
  return launch_status("cache_append_kernel");
}
