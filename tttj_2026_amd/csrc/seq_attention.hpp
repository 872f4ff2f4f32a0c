// Attention of ragged token rows: whole prompts packed one behind the other (keys in rows of their own), and new
// tokens over a paged cache.  Device code of seq_attention.hip and seq_attention_wide.hip.
//
//   o_i = sum_{j < lim_i} exp(c q_i.k_j - m_i) v_j / sum_{j < lim_i} exp(c q_i.k_j - m_i)
//
// with lim_i the keys that token i may see (its own position + 1, or all of its sequence's).  Query heads share
// key / value heads in groups of G: a row of the problem is a (token, head of the group) pair, G rows per token,
// so one tile of K and V serves all heads of its group, and the rows of a tile span few tokens, which keeps the
// part of a causal tile that is computed and masked small.
//
// A block takes tiles of 32 RW rows of one (sequence, kv head), and of each all keys or a range.  Its waves form KW groups
// of RW: the waves of a group share key tiles of KT keys, staged in LDS two deep, and each owns 32 rows; the groups
// take alternate tiles and are joined through LDS at the end.
// * RW 4, KW 1, KT 64 (wide: prompts and chunks).  Bound by the matrix unit and the vector instructions of the softmax
//   beside it: one 32x32x16 product leaves room for about four of them, and 5.6 to 8 are needed (heads of 128).  The exps
//   of 32 keys run beside the products Q K^T of the next 32, so K is staged 32 keys ahead of V.
// * RW 1, KT 32, KW 2 (narrow; 1 above heads of 128) and, where blocks are few, KW 8 / 4 / 2 (deep; heads to 64 / 128 /
//   256): single tokens and drafts.  Bound by HBM: every wave streams tiles of its own without a barrier, close to two
//   in flight.  KW 1 / 2 / 4 for 64 tokens over 1 to 4000 keys on 8 heads of 128: 130 / 108 / 117 us.
// How tiles are given to blocks: kSeq... below.  Where a tile's keys are split over blocks, parts of O with a maximum and
// a sum each go through a workspace, and the seq_merge kernels join them.
//
// Measured on MI355X: prompts of 8192 and 3130 tokens, causal, 32 heads of 128 on 8, bf16: 576 us, 1.09 PFLOP/s (matrix
// unit 57% busy, vector units 47%, one of them 82%, at 1.80 GHz); 2 x 4096 tokens on 16 heads of 64 87 us, 0.79 PFLOP/s;
// 12 prompts of 85 to 1500 tokens 113 us, 0.70 (a block takes 7 us to start and end, 1.8 us a tile of keys); 4 x 4096 on 16
// heads of 256 631 to 650 us, 0.85 PFLOP/s; 512 new tokens each for 8 sequences of up to 4608 keys 184 us, 0.89 PFLOP/s (2.1
// us a tile: pages are looked up beside it).  4 tokens over 100000 keys each, 8 heads of 128: 287 us, 5.7 TB/s; 64 over 1 to
// 4000: 106 us.
//
// The cache may be in 8 bits (C8): e4m3 and a power of two for each block of tokens and head, widened to T by one instruction
// per two values.  Narrow blocks copy the bytes into LDS, in tiles of 64 keys on heads to 128, and 2 or 4 of their waves share
// a tile, each for a head of its own, where heads lie side by side: pieces of 64, 128, 256 and 512 bytes a row are read at
// 3.0, 5.5, 6.0 and 6.2 TB/s.  64 tokens over 8000 keys, 32 heads of 128 on 8, bf16: 195 us, 5.4 TB/s; over lengths of 67 to 8000
// 107 us, 4.9; 64 over 4000 keys on 16 heads of 64 105 us, 5.0; 4 over 100000 on 64 heads of 128 on 8 154 us, 5.3.  8 chunks of
// 512 over up to 4608 keys 196 to 203 us, 0.84 to 0.81 PFLOP/s (16 bits: 183; 32 of 280 vector instructions a tile widen, and
// 10 more find the scales).
//
// Per wave and tile: S^T = K Q^T with v_mfma_f32_32x32x16 (lane l holds row l % 32; of its 32 keys per block those
// with bit 2 equal to l / 32), softmax with a running maximum and sum in fp32, O^T += V^T P^T.  K and V stay in the
// row-major form of the projections and of the cache: ds_read_b64_tr_b16 transposes V on its way from LDS, and reads
// the keys in the order in which a lane holds its probabilities, so neither needs a shuffle.
// Scores are multiplied by c log2(e) in fp32 (rounding q c to 16 bits would cost as much precision as rounding the
// probabilities does).  Probabilities are rounded to the type of V for the matrix unit, relative to a maximum that
// is moved only when it grows by more than 2^8 (lazy rescaling), and times 2^7 in fp16, which so holds what is down to
// 2^-31 of the largest: 100000 keys of 2^-25 each still count; times 2^-24 in bf16, whose values go up to 2^128 and would
// overflow the sums (its probabilities go down to 2^-102 of the largest).
#pragma once

#include "attention_block.hpp"

#include <type_traits>

#define TT_INLINE __attribute__((always_inline))

namespace tt {

using bf16 = __bf16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Num;
template <>
struct Num<half> {
  using v2 = half2v;
  using v8 = half8;
  static constexpr uint16_t kExp = 0x7c00;  // the exponent's bits: all set in infinities and NaN
  static constexpr float kShift = 7.f;      // log2 of the factor on the probabilities (kSeqLazy): 2^(8 + 7) < 65504
  static __device__ __forceinline__ floatx16 mfma(v8 a, v8 b, floatx16 c) { return mfma32x32x16(a, b, c); }
  static __device__ __forceinline__ float add2(v2 p, float c) {
    return __builtin_amdgcn_fdot2(p, v2{(half)1.f, (half)1.f}, c, false);
  }
  static constexpr int kTop = 127 + 7;  // above this scale (as e8m0) the largest of e4m3, 448, lies past the type's
  template <bool HI>
  static __device__ __forceinline__ uint32_t widen(uint32_t x, float scale) {  // bytes 0, 1 (2, 3) of e4m3
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, HI));
  }
};
template <>
struct Num<bf16> {
  using v2 = bf16x2;
  using v8 = bf16x8;
  static constexpr uint16_t kExp = 0x7f80;
  static constexpr float kShift = -24.f;  // 65536 keys of 2^(8 - 24) times the largest value do not overflow fp32
  static __device__ __forceinline__ floatx16 mfma(v8 a, v8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(v2 p, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(p, v2{(bf16)1.f, (bf16)1.f}, c, false);
  }
  static constexpr int kTop = 127 + 119;
  template <bool HI>
  static __device__ __forceinline__ uint32_t widen(uint32_t x, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, HI));
  }
};

// Eight values of an 8-bit cache in T: e4m3 times a power of two, the bits of an e8m0 as an exponent (exact wherever T
// holds the product; past T's largest they are infinities).
template <typename T>
__device__ __forceinline__ u32x4 widen8(u32x2 x, float scale) {
  return u32x4{Num<T>::template widen<false>(x[0], scale), Num<T>::template widen<true>(x[0], scale),
               Num<T>::template widen<false>(x[1], scale), Num<T>::template widen<true>(x[1], scale)};
}
__device__ __forceinline__ float e8m0(uint32_t e) { return __builtin_bit_cast(float, e << 23); }

// The smallest magnitude of e4m3 (7 bits) that is no number or, times 2^(e - 127), past T's largest.
template <typename T>
__device__ __forceinline__ uint32_t widen_limit(int e) {
  const int over = e - Num<T>::kTop - 1;  // 2^(8 - over) and above lie past it
  if (over < 0) return 0x7f;
  return over <= 14 ? 0x78 - 8 * over : 1 << max(17 - over, 0);  // (below 2^-6 e4m3 counts in steps of 2^-9)
}

// ds_read_b64_tr_b16 (16 lanes transpose their 4 rows of 16).  The __restrict gives the read alias information;
// without any, the compiler lets it wait for every global -> LDS copy in flight.
using lds_short = __attribute__((address_space(3))) short;
__device__ __forceinline__ shortx4 read_tr16(const lds_short* __restrict__ p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4*)p);
}

// ds_read_b64_tr_b8: 16 lanes transpose their 8 rows of 16 bytes.
__device__ __forceinline__ u32x2 read_tr8(const lds_short* __restrict__ p) {
  typedef int intx2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) intx2*)p));
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const lds_short*)p;
}

__device__ __forceinline__ void lds_done() {  // this wave's LDS accesses, its copies in flight apart
  __builtin_amdgcn_s_waitcnt(0xC07F);
  asm volatile("" ::: "memory");
}

struct SeqAttnArgs {
  const void *q, *k, *v;   // q rows [tokens, heads, head_dim]; k, v the same with kv_heads, or a paged cache
  void* out;               // [tokens, heads * head_dim]
  const int32_t* starts;   // [batch + 1] first row of each sequence; nullptr: row b is sequence b
  const int32_t* lengths;  // cache: keys of each sequence, its new tokens among them
  const int32_t* table;    // cache: page numbers, table_row apart, table_pages of them per sequence
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  int64_t k_page, v_page, table_row;
  int tokens, batch, heads, kv_heads, group, head_dim;
  int pages, table_pages, page_shift;
  int causal;
  float scale_log2;        // c log2(e)
  int slots;               // blocks of the launch per kv head
  int mode;                // kSeqInOrder, kSeqHeaviest or kSeqShares
  float* part_o;           // kSeqShares: [2 slots][kv_heads][R * head_dim], the rows of tiles that lie in several shares
  float2* part_ml;         // ... [2 slots][kv_heads][R], their maximum (log2 domain) and sum
  // 8-bit cache: the exponents (e8m0) of k and v, one per 2^block_shift tokens of a page and head; strides in bytes, of both
  // (an offset has 32 bits).
  const uint8_t *k_scale, *v_scale;
  int s_page, s_block, s_head;
  int block_shift;
};

// Where feature d of row r of a tile lies in a part of 128 rows: as the lanes hold them, 32 rows x 8 features in turn, so
// that every store is one run of 1 KiB (in rows of features, where a store touches 32 rows, 16 chunks of 128 rows on heads
// of 256 over 4096 keys took 33 us + 10 to join; so 29 + 8).
__device__ __forceinline__ int wide_place(int head_dim, int r, int d) {
  return (((r >> 5) * (head_dim >> 3) + (d >> 3)) * 64 + ((d >> 2) & 1) * 32 + (r & 31)) * 4 + (d & 3);
}

// How row tiles are given to blocks.
constexpr int kSeqInOrder = 0;   // a tile each, the last sequence's last tile first
constexpr int kSeqHeaviest = 1;  // a tile each, those with most keys first, over all sequences (batch <= 64)
constexpr int kSeqShares = 2;    // all (tile, 64 keys) units of a kv head in equal shares, one per block
constexpr int kSeqUnit = 64;
constexpr int kSeqLevels = 32;
constexpr int kSeqMinShare = 4;  // units (4 / 6 / 8 / 12: chunks of 3 prompts on heads of 256 37.7 / 42 / 45.6 / 57 us)
constexpr int kSeqTileCost = 2;  // units that a tile's beginning and end take the time of (0 / 2 / 4: the same chunks 45.8
                                 // / 38.6 / 39.5 us, 64 tokens over 1 to 4000 keys 106.6 / 105 / 107)

constexpr float kSeqLazy = 8.0f;   // log2 growth of a row's maximum that moves its reference

// exp2 of a difference of maxima, as the weight of sums that are joined: never 0, so that an infinity among them stays one
// (2^-149, for less than 2^-126, of any finite sum is below half a step of the others).
__device__ __forceinline__ float seq_weight(float log2) {
  return fmaxf(__builtin_amdgcn_exp2f(log2), 0x1p-149f);
}

// V tiles are read by ds_read_b64_tr_b16: half a wave reads 64 bytes of each of 4 consecutive rows.  The 64-byte
// segments of a row are exchanged by its number so that those 4 pieces lie in different quarters of the 64 banks.
template <int HD>
__device__ __forceinline__ int vseg(int row, int c) {
  if constexpr (HD >= 128) return c ^ ((row & 3) << 2);
  else if constexpr (HD == 64) return c ^ ((row & 2) << 1);
  else return c;
}

// The same for tiles of an 8-bit cache, whose LDS rows are HD bytes in chunks of 16.  K: 16 lanes read one chunk of 16
// rows.  V: 16 lanes read one chunk of rows 4 h ... 4 h + 3 and 8 further, and 16 others the next chunk.
template <int HD>
__device__ __forceinline__ int kswz8(int row, int c) {
  if constexpr (HD == 256) return c ^ (row & 15);
  else if constexpr (HD == 128) return c ^ ((row >> 1) & 7);
  else return c ^ ((row >> 2) & 3);
}
template <int HD>
__device__ __forceinline__ int vseg8(int row, int c) {
  if constexpr (HD == 256) return c ^ ((row & 3) << 1 | (row & 8));
  else if constexpr (HD == 128) return c ^ ((row & 2) | ((row & 8) >> 1));
  else return c ^ ((row & 8) >> 2);
}

// Tiles of T that are widened on their way into LDS: a lane writes two chunks, 2 c and 2 c + 1, and 8 lanes at a time 128
// bytes without conflict if the even chunks of a row come first and the odd ones behind them (and with rows of 128 bytes,
// halves of odd rows change places).  Reads as of the other tiles.  (8 chunks of 512: 2 us of 198.)
template <int HD>
__device__ __forceinline__ int kswz_widened(int row, int c) {
  const int p = c >> 1 | (c & 1) << (HD == 128 ? 3 : 2);
  return HD == 128 ? p ^ (row & 15) : p ^ ((row >> 1) & 7) ^ ((row & 1) << 2);
}
template <int HD>
__device__ __forceinline__ int vseg_widened(int row, int c) {
  const int p = c >> 1 | (c & 1) << (HD == 128 ? 3 : 2);
  return HD == 128 ? p ^ ((row & 3) << 1) : p ^ ((row & 2) | (row & 1) << 2);
}

// The sequence that owns row tile `slot`.  Sequence b's tiles start at slot floor(starts[b] G / R) + b, which
// leaves it at least as many as it has, and no table of tiles is needed; the search takes 64 candidates a step.
struct SeqTile {
  int seq, tile, first, count;  // the sequence, its row tile, its first row and its rows
};

__device__ __forceinline__ int seq_start(const int32_t* starts, int b, int tokens) {
  return min(max(starts[b], 0), tokens);
}

template <class Key>
__device__ __forceinline__ int seq_search(int batch, int at, Key key) {  // the last b with key(b) <= at (0: none)
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) >> 6;
    const int b = lo + lane * step;
    const int n = __popcll(__ballot(b < hi && key(min(b, batch - 1)) <= at));
    lo += max(n - 1, 0) * step;
    hi = min(hi, lo + step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

__device__ __forceinline__ SeqTile seq_tile(const SeqAttnArgs& a, int slot, int rows_per_tile) {
  SeqTile s;
  if (a.starts == nullptr) {
    const int tiles = (a.group + rows_per_tile - 1) / rows_per_tile;
    s.seq = slot / tiles;
    s.tile = slot - s.seq * tiles;
    s.first = s.seq;
    s.count = 1;
    return s;
  }
  const auto slot_of = [&](int b) { return seq_start(a.starts, b, a.tokens) * a.group / rows_per_tile + b; };
  s.seq = seq_search(a.batch, slot, slot_of);
  s.tile = slot - slot_of(s.seq);
  s.first = seq_start(a.starts, s.seq, a.tokens);
  s.count = seq_start(a.starts, s.seq + 1, a.tokens) - s.first;
  return s;
}

// First row and rows of sequence b.
__device__ __forceinline__ int2 seq_rows(const SeqAttnArgs& a, int b) {
  if (a.starts == nullptr) return make_int2(b, 1);
  const int first = seq_start(a.starts, b, a.tokens);
  return make_int2(first, max(seq_start(a.starts, b + 1, a.tokens) - first, 0));
}

// Keys that sequence `seq` of `count` rows holds.
template <bool PAGED>
__device__ __forceinline__ int seq_keys(const SeqAttnArgs& a, int seq, int count) {
  if constexpr (PAGED) return min(max(a.lengths[seq], 0), a.table_pages << a.page_shift);
  else return count;
}

// Keys that token i of `count` may see, of `keys`.
__device__ __forceinline__ int seq_limit(const SeqAttnArgs& a, int i, int count, int keys) {
  return a.causal ? max(keys - count + i + 1, 0) : keys;
}

// Sum over the lanes up to this one, by DPP: shifts by 1, 2, 4 and 8 within rows of 16 lanes, then the last lane of
// row 0 (2) to row 1 (3) and that of row 1 to rows 2 and 3.
__device__ __forceinline__ int wave_scan_int(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

__device__ __forceinline__ int wave_sum_int(int v) { return __builtin_amdgcn_readlane(wave_scan_int(v), 63); }

__device__ __forceinline__ int wave_max_int(int v) {  // of values >= 0
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(v, 63);
}

// The tile of rank `rank` by its number of keys (kSeqHeaviest; lane b holds sequence b): the tiles of a sequence that
// see more than w units of keys are those from a certain one on, so their number over all sequences follows from w
// without a list, and a bisection over w finds the rank's level.  A unit is a 32nd of the most keys; within a
// level, tiles go sequence by sequence.  tile < 0: no such tile.
template <bool PAGED>
__device__ __forceinline__ SeqTile seq_ranked(const SeqAttnArgs& a, int rank, int rows_per_tile) {
  const int lane = threadIdx.x & 63, G = a.group;
  int2 own = make_int2(0, 0);
  int keys = 0;
  if (lane < a.batch) {
    own = seq_rows(a, lane);
    keys = seq_keys<PAGED>(a, lane, own.y);
  }
  const int tiles = (own.y * G + rows_per_tile - 1) / rows_per_tile;
  const int unit = (wave_max_int(keys) + kSeqLevels - 1) / kSeqLevels;
  // The first tile with a row that sees more than w units of keys (w < 0: any row).
  const auto from = [&](int w) -> int {
    if (w < 0) return 0;
    if (!a.causal) return keys > unit * w ? 0 : tiles;
    const int token = unit * w - (keys - own.y);
    return token <= 0 ? 0 : token >= own.y ? tiles : token * G / rows_per_tile;
  };
  SeqTile s{0, -1, 0, 0};
  if (rank >= wave_sum_int(tiles)) return s;
  int lo = -1, hi = kSeqLevels;  // more than `rank` tiles above lo, not above hi
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (wave_sum_int(tiles - from(mid)) > rank) lo = mid;
    else hi = mid;
  }
  const int at = rank - wave_sum_int(tiles - from(lo + 1));  // among the tiles of this level
  const int here = from(lo + 1) - from(lo);
  const int upto = wave_scan_int(here);
  const int b = __ffsll((unsigned long long)__ballot(upto > at)) - 1;
  s.seq = __builtin_amdgcn_readfirstlane(b);
  s.tile = __builtin_amdgcn_readlane(from(lo) + at - (upto - here), s.seq);
  s.first = __builtin_amdgcn_readlane(own.x, s.seq);
  s.count = __builtin_amdgcn_readlane(own.y, s.seq);
  return s;
}

// kSeqShares.  A sequence counts tiles x units units: kSeqTileCost, which hold no keys, and its keys in units of 64 (at
// least one), whether or not all rows of a tile see them (its new tokens are few against its keys wherever keys are
// shared out).  A tile's parts are the shares that hold keys of it.
struct SeqUnits {
  int first, count, keys, tiles, units;
};

__device__ __forceinline__ SeqUnits seq_units(const SeqAttnArgs& a, int b, int rows_per_tile) {
  SeqUnits u;
  const int2 own = seq_rows(a, b);
  u.first = own.x;
  u.count = own.y;
  u.keys = seq_keys<true>(a, b, own.y);
  u.tiles = (own.y * a.group + rows_per_tile - 1) / rows_per_tile;
  u.units = max((u.keys + kSeqUnit - 1) / kSeqUnit, 1) + kSeqTileCost;
  return u;
}

struct SeqShare {
  int total, share;  // units of a kv head, and those of one block
  int seq, base;     // the sequence asked for, and its first unit
  SeqUnits units;
};

// The shares of a launch, and the sequence that holds the first unit of block `slot` (seq < 0), or sequence `seq`.  Where
// `starts` falls anywhere, rows belong to several sequences and the units have no bound: there are none (total 0).
__device__ __forceinline__ SeqShare seq_share(const SeqAttnArgs& a, int slot, int seq, int rows_per_tile) {
  const int lane = threadIdx.x & 63;
  bool falls = false;
  const auto units_of = [&](int b) -> SeqUnits {
    if (b >= a.batch) return SeqUnits{0, 0, 0, 0, 1};
    falls |= a.starts != nullptr && seq_start(a.starts, b, a.tokens) > seq_start(a.starts, b + 1, a.tokens);
    return seq_units(a, b, rows_per_tile);
  };
  SeqShare s;
  SeqUnits u = units_of(lane);
  int upto = wave_scan_int(u.tiles * u.units);
  s.total = __builtin_amdgcn_readlane(upto, 63);
  if (a.batch > 64) {
    int n = 0;
    for (int b = 64 + lane; b < a.batch; b += 64) {
      const SeqUnits v = units_of(b);
      n += v.tiles * v.units;
    }
    s.total += wave_sum_int(n);
  }
  if (__builtin_amdgcn_ballot_w64(falls) != 0) s.total = 0;
  s.share = max((s.total + a.slots - 1) / a.slots, kSeqMinShare);
  const int64_t x = (int64_t)slot * s.share;
  s.base = 0;
  for (int b0 = 0;;) {
    const int all = __builtin_amdgcn_readlane(upto, 63);
    if (b0 + 64 >= a.batch || (seq >= 0 ? seq < b0 + 64 : s.base + all > x)) {
      const int l = min(seq >= 0 ? seq - b0 : __popcll(__ballot(s.base + upto <= x)), 63);
      s.seq = b0 + l;
      if (l > 0) s.base += __builtin_amdgcn_readlane(upto, l - 1);
      s.units = SeqUnits{__builtin_amdgcn_readlane(u.first, l), __builtin_amdgcn_readlane(u.count, l),
                         __builtin_amdgcn_readlane(u.keys, l), __builtin_amdgcn_readlane(u.tiles, l),
                         __builtin_amdgcn_readlane(u.units, l)};
      return s;
    }
    s.base += all;
    b0 += 64;
    u = units_of(b0 + lane);
    upto = wave_scan_int(u.tiles * u.units);
  }
}

template <typename T, int HD, int RW, int KW, int KT, bool PAGED, bool C8 = false, int NH = 1,
          int WPE = C8 && RW == 1 ? (HD <= 64 ? 2 : 1) : (HD <= 64 ? 3 : HD <= 128 ? 2 : 1)>
__global__ __launch_bounds__(64 * RW * KW * NH) __attribute__((amdgpu_waves_per_eu(WPE, WPE))) void seq_attention_kernel(SeqAttnArgs a) {
  using v2 = typename Num<T>::v2;
  using v8 = typename Num<T>::v8;
  constexpr int R = 32 * RW;                // rows of a block (64 a wave leave registers for one wave per SIMD only)
  constexpr bool PIPE = RW > 1;              // softmax beside the next keys' products
  constexpr int KSTEPS = HD / 16;           // k-steps of S^T
  constexpr int DB = HD / 32;               // 32-row blocks of O^T
  constexpr int CH = HD / 8;                // 16-byte chunks of a row of T
  constexpr int RPC = 64 / CH;              // rows of T in 1 KiB
  // An 8-bit cache's tiles: narrow blocks copy their bytes, and a wave widens the fragments that it reads.  In wide ones each
  // row is widened once for all waves: its bytes are copied to a place of the wave's own behind the tiles, and from there
  // they go through registers into the tile as T, beside the products of the last step before it (8 chunks of 512 tokens:
  // 212 us behind that step, 201 beside it; 200 with the bytes on their way in registers, 16 more than there are, some
  // of which then lie in scratch memory).
  constexpr bool RAW = C8 && !PIPE;
  using E = std::conditional_t<RAW, uint8_t, T>;
  constexpr int EB = C8 ? 1 : 2;            // bytes of a value in memory
  // NH waves of a block over an 8-bit cache share its tiles, each for a head of its own: HD bytes are less than memory is
  // best read in.
  static_assert(NH == 1 || (RAW && KW == 1), "heads side by side");
  constexpr int ROW = NH * HD;              // values of a row of a tile
  constexpr int CB = ROW * EB / 16;         // 16-byte chunks of a row in memory
  constexpr int RPB = 64 / CB;              // rows per 1 KiB copy
  constexpr int WROWS = KT / (RW * NH);     // rows of a tile that one wave copies
  constexpr int PG = WROWS / 16;            // ... in groups of 16, each of which lies in one page
  constexpr int CPG = 16 / RPB;             // copies per group
  constexpr int TILE = KT * ROW;
  static_assert(WROWS % 16 == 0 && RPB <= 16, "a wave copies whole 16-row groups");
  static_assert(!C8 || (PAGED && HD >= 64), "8 bits: a cache");

  extern __shared__ __align__(512) char seq_lds[];

  const int slot = blockIdx.x / (a.kv_heads / NH);
  const int G = a.group;
  const int tid = threadIdx.x;
  int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = RW == 1 ? 0 : wave % RW, grp = NH > 1 ? 0 : RW == 1 ? wave : wave / RW;
  const int hw = NH > 1 ? wave : 0, cw = NH > 1 ? hw : rw;  // this wave's head of the block's; its rows of a copied tile
  const int hkv0 = blockIdx.x % (a.kv_heads / NH) * NH, hkv = hkv0 + hw;
  int hf = lane >> 5, col = lane & 31;
  E* const sk = reinterpret_cast<E*>(seq_lds) + (size_t)grp * 2 * TILE;
  E* const sv = reinterpret_cast<E*>(seq_lds) + (size_t)KW * 2 * TILE + (size_t)grp * 2 * TILE;

  // What this block does: a row tile with all its keys, or (kSeqShares) units x ... share_end - 1, tile after tile.
  SeqTile sq;
  const bool shares = PAGED && a.mode == kSeqShares;
  int x = 0, share_end = 0, base = 0;
  SeqUnits su{};
  if (shares) {
    const SeqShare sh = seq_share(a, slot, -1, R);
    if ((int64_t)slot * sh.share >= sh.total) return;
    x = slot * sh.share;
    share_end = min(sh.total - x, sh.share) + x;
    sq.seq = sh.seq;
    base = sh.base;
    su = sh.units;
  } else {
    if (a.mode == kSeqHeaviest) sq = seq_ranked<PAGED>(a, slot, R);
    else sq = seq_tile(a, a.slots - 1 - slot, R);
    if (sq.tile < 0 || sq.tile * R >= sq.count * G) return;
  }

  // Copy sources: lane l of copy c of a group fetches row c RPB + l / CB of the group into the next 16 bytes of
  // LDS, from the chunk that belongs there.  Chunks at or past head_dim lie outside the buffer: LDS keeps the zeros
  // that it is cleared to (or receives those that such a load returns).
  const int hd = a.head_dim;
  uint32_t koff[CPG], voff[CPG];
#pragma unroll
  for (int c = 0; c < CPG; ++c) {
    const int row = c * RPB + lane / CB;
    int kc = lane % CB, vc = lane % CB;
    if constexpr (RAW) kc = kswz8<ROW>(row, kc) * 16, vc = vseg8<ROW>(row, vc) * 16;
    else if constexpr (C8) kc *= 16, vc *= 16;
    else kc = kswz<HD>(row, kc) * 8, vc = vseg<HD>(row, vc) * 8;
    if constexpr (NH > 1) {  // head_dim values of each head
      const int k_at = kc / HD * (int)a.k_head + kc % HD, v_at = vc / HD * (int)a.v_head + vc % HD;
      koff[c] = kc % HD < hd ? (uint32_t)(row * (int)a.k_row + k_at) : 0x80000000u;
      voff[c] = vc % HD < hd ? (uint32_t)(row * (int)a.v_row + v_at) : 0x80000000u;
      continue;
    }
    koff[c] = kc < hd ? (uint32_t)(row * (int)a.k_row + kc) * EB : 0x80000000u;
    voff[c] = vc < hd ? (uint32_t)(row * (int)a.v_row + vc) * EB : 0x80000000u;
  }
  using Mem = std::conditional_t<C8, uint8_t, T>;
  const Mem* const kh = static_cast<const Mem*>(a.k) + hkv0 * a.k_head;
  const Mem* const vh = static_cast<const Mem*>(a.v) + hkv0 * a.v_head;

  const float c2 = a.scale_log2, lazy = kSeqLazy / a.scale_log2;
  // LDS addresses of this lane's pieces of the first K and V block of a stage; the others lie at constant distances.
  // (The empty asm keeps each in one register: the compiler would spread the sums over many.)  Rows of 512 bytes
  // leave no registers for them: there the pieces of a row are told apart by an XOR of the first one's address.
  constexpr bool FAR = PIPE && HD > 128;
  // Whether a tile's bytes are widened beside the products of the last step before it (heads above 128: after it).
  constexpr bool BESIDE = C8 && PIPE && !FAR;
  constexpr int KA = FAR ? 1 : RAW ? KSTEPS / 2 : KSTEPS, VA = FAR ? 1 : DB;
  uint32_t kread[KA], vread[VA];
#pragma unroll
  for (int kk = 0; kk < KA; ++kk) {
    if constexpr (RAW) kread[kk] = lds_address(sk + col * ROW + kswz8<ROW>(col, hw * HD / 16 + 2 * kk + hf) * 16);
    else kread[kk] = lds_address(sk + col * HD + (BESIDE ? kswz_widened<HD>(col, 2 * kk + hf) : kswz<HD>(col, 2 * kk + hf)) * 8);
    asm volatile("" : "+v"(kread[kk]));
  }
  // (RAW: 16 lanes read 8 rows, 4 hf ... 4 hf + 3 and 8 further, in the order of the lane's probabilities)
  const int vrow = RAW ? 4 * hf + ((lane >> 1) & 3) + (lane & 8) : 4 * hf + ((lane >> 2) & 3);
#pragma unroll
  for (int i = 0; i < VA; ++i) {
    if constexpr (RAW) {
      const int c = hw * HD / 16 + 2 * i + ((lane >> 4) & 1);
      vread[i] = lds_address(sv + vrow * ROW + vseg8<ROW>(vrow, c) * 16 + 8 * (lane & 1));
    } else {
      int c = 4 * i + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
      c = BESIDE ? vseg_widened<HD>(vrow, c) : vseg<HD>(vrow, c);
      vread[i] = lds_address(sv + vrow * HD + c * 8 + 4 * (lane & 1));
    }
    asm volatile("" : "+v"(vread[i]));
  }
  for (;;) {
  // (What follows from these is worked out again for each tile instead of being held in registers throughout.)
  asm volatile("" : "+v"(lane), "+v"(hf), "+v"(col));
  if (hd < HD) {  // the tile before left its sums or rows there
    constexpr int BEHIND = C8 && PIPE ? RW * 2 * CPG * 1024 : 0;  // bytes on their way into the tiles
    for (int e = tid; e < (4 * KW * TILE * (int)sizeof(E) + BEHIND) / 16; e += 64 * RW * KW * NH)
      reinterpret_cast<u32x4*>(seq_lds)[e] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
  }
  int keys, kbeg = 0, kend = INT32_MAX, part = -1;
  if (shares) {
    while (x >= base + su.tiles * su.units) {  // the next sequence that has rows
      if (sq.seq + 1 >= a.batch) return;
      base += su.tiles * su.units;
      su = seq_units(a, ++sq.seq, R);
    }
    sq.first = su.first;
    sq.count = su.count;
    sq.tile = (x - base) / su.units;
    keys = su.keys;
    const int begin = x - base - sq.tile * su.units, end = min(begin + share_end - x, su.units);
    x += end - begin;
    if (end <= kSeqTileCost) return;  // nothing but a tile's beginning was left of the share
    const bool first = begin <= kSeqTileCost;
    if (!first) kbeg = (begin - kSeqTileCost) * kSeqUnit;
    if (end < su.units) kend = (end - kSeqTileCost) * kSeqUnit;
    if (!first || end < su.units) part = 2 * slot + (first ? 1 : 0);
  } else {
    keys = seq_keys<PAGED>(a, sq.seq, sq.count);
  }
  const int rows = sq.count * G;
  const int r0 = sq.tile * R;
  const int block_end = seq_limit(a, min(r0 + R - 1, rows - 1) / G, sq.count, keys);
  kend = min(kend, block_end);
  const int ntiles = kend > kbeg ? (kend - kbeg + KT - 1) / KT : 0;

  // Rows of this wave; those behind the last repeat it and are not stored, so limits rise along the rows.
  const int wr0 = r0 + rw * 32;
  const bool wave_active = wr0 < rows;
  const int block_lo = seq_limit(a, r0 / G, sq.count, keys);  // the first row's
  const int lim_lo = seq_limit(a, min(wr0, rows - 1) / G, sq.count, keys);
  const int lim_hi = min(seq_limit(a, min(wr0 + 31, rows - 1) / G, sq.count, keys), kend);
  const int own = min(wr0 + col, rows - 1);  // this lane's row
  const int tok = own / G, head = hkv * G + own - tok * G, lim = seq_limit(a, tok, sq.count, keys);

  // Paged: lane l holds the page of the 16-key group l behind key t0 (of the first 8).
  auto tile_pages = [&](int t0) TT_INLINE -> int {
    const int key = min(t0 + 16 * (lane & 7), max(keys - 1, 0));
    return a.table[sq.seq * a.table_row + (key >> a.page_shift)];
  };
  // Which of those lie outside the cache (a bit each); their keys are not read (place: no bytes there) and count as NaN.
  // Rows that do not see them multiply whatever the tile then holds in V by 0 as they do other values (settle_v).
  auto bad_groups = [&](int pe, int t0) TT_INLINE -> uint32_t {
    return (uint32_t)__ballot((uint32_t)pe >= (uint32_t)a.pages && t0 + 16 * lane < keys) & 0xffu;
  };
  // 8 bits: the scales of those groups (blocks of tokens hold whole groups), as they are loaded: whatever is done with them
  // waits for them.  A group one of whose scales is none (255) counts as one outside the cache; its V is multiplied by
  // 2^-127.
  struct Scales {
    uint8_t k, v;
  };
  auto tile_scales = [&](int pe, int t0) TT_INLINE -> Scales {
    const uint32_t in = min(t0 + 16 * (lane & 7), max(keys - 1, 0)) & ((1 << a.page_shift) - 1);
    const uint32_t page = (uint32_t)pe < (uint32_t)a.pages ? pe : 0, block = in >> a.block_shift;
    const uint32_t at = page * (uint32_t)a.s_page + block * (uint32_t)a.s_block + (uint32_t)(hkv * a.s_head);
    return Scales{a.k_scale[at], a.v_scale[at]};
  };
  auto bad_scales = [&](const Scales& se, int t0) TT_INLINE -> uint32_t {
    return (uint32_t)__ballot((se.k == 255 || se.v == 255) && t0 + 16 * lane < keys) & 0xffu;
  };
  auto scale_of = [&](const Scales& se, int group, bool is_k) TT_INLINE -> float {
    const uint32_t e = __builtin_amdgcn_readlane(is_k ? se.k : se.v, group) & 255;
    return e8m0(e == 255 ? 0 : e);
  };
  // Where those groups lie in K and V (bytes), and how many bytes there belong to keys; worked out by the lanes for
  // pages, whose numbers they hold, and by the scalar unit otherwise.
  struct Places {
    uint64_t k, v;
    uint32_t k_bytes, v_bytes;
  };
  auto place = [&](int t, int pe) TT_INLINE -> Places {
    int n = min(max(keys - t, 0), 16);
    Places p;
    if constexpr (PAGED) {
      if ((uint32_t)pe >= (uint32_t)a.pages) n = pe = 0;
      const uint32_t page = pe, in = t & ((1 << a.page_shift) - 1);
      p.k = EB * (page * (uint64_t)a.k_page + in * (uint64_t)a.k_row);
      if (C8 && a.k_page == a.v_page && a.k_row == a.v_row) p.v = p.k;  // (half of eight long multiplications)
      else p.v = EB * (page * (uint64_t)a.v_page + in * (uint64_t)a.v_row);
    } else {
      const uint32_t row = sq.first + min(t, keys - 1);
      p.k = 2 * (row * (uint64_t)a.k_row);
      p.v = 2 * (row * (uint64_t)a.v_row);
    }
    p.k_bytes = n == 0 ? 0 : EB * ((n - 1) * (uint32_t)a.k_row + (NH - 1) * (uint32_t)a.k_head + hd);
    p.v_bytes = n == 0 ? 0 : EB * ((n - 1) * (uint32_t)a.v_row + (NH - 1) * (uint32_t)a.v_head + hd);
    return p;
  };
  auto places = [&](int pe, int t0) TT_INLINE -> Places {
    if constexpr (PAGED) return place(t0 + 16 * (lane & 7), pe);
    else return Places{(uint64_t)t0, 0, 0, 0};
  };
  // Copies of this wave's rows of a K (V) tile whose first 16 keys are group `group` of `at`, to `tile` (wide blocks, 8
  // bits: their bytes to `bytes`, from where write_half takes them into the tile).
  auto issue_half = [&](bool is_k, const Places& at, E* tile, int group, char* bytes = nullptr) TT_INLINE {
#pragma unroll
    for (int p = 0; p < PG; ++p) {
      const int g = cw * PG + p;
      if (group + g < 0) continue;
      uint64_t where;
      uint32_t size;
      if constexpr (PAGED) {
        const uint64_t w = is_k ? at.k : at.v;
        where = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(w >> 32), group + g) << 32 |
                (uint32_t)__builtin_amdgcn_readlane((int)w, group + g);
        size = __builtin_amdgcn_readlane((int)(is_k ? at.k_bytes : at.v_bytes), group + g);
      } else {
        const Places q = place((int)at.k + 16 * (group + g), 0);
        where = is_k ? q.k : q.v;
        size = is_k ? q.k_bytes : q.v_bytes;
      }
      const __amdgpu_buffer_rsrc_t r = buffer_rsrc(reinterpret_cast<const char*>(is_k ? kh : vh) + where, size);
#pragma unroll
      for (int c = 0; c < CPG; ++c) {
        half* const to = reinterpret_cast<half*>(tile + (g * 16 + c * RPB) * ROW);
        lds_copy16_buf(r, is_k ? koff[c] : voff[c], C8 && PIPE ? reinterpret_cast<half*>(bytes + c * 1024) : to);
      }
    }
  };
  char* const k_bytes = seq_lds + 4 * TILE * sizeof(T) + (size_t)rw * 2 * CPG * 1024;  // wide, 8 bits
  char* const v_bytes = k_bytes + CPG * 1024;
  using Bytes = u32x4[CPG];
  auto read_bytes = [&](Bytes& x, const char* bytes) TT_INLINE {
#pragma unroll
    for (int c = 0; c < CPG; ++c) x[c] = *reinterpret_cast<const u32x4*>(bytes + c * 1024 + lane * 16);
  };
  auto write_half = [&](bool is_k, const Scales& se, E* tile, int group, const Bytes& x) TT_INLINE {
    if constexpr (C8 && PIPE) {
      static_assert(PG == 1, "a group per wave");
      if (group < 0 && group + rw < 0) return;
      const float scale = scale_of(se, group + rw, is_k);
#pragma unroll
      for (int c = 0; c < CPG; ++c) {
        const int row = rw * 16 + c * RPB + lane / CB, chunk = 2 * (lane % CB);
        T* const to = tile + row * HD;
        int at, next = 1;  // where the chunk lies, and what its place and the next chunk's differ by
        if constexpr (BESIDE) {
          at = is_k ? kswz_widened<HD>(row, chunk) : vseg_widened<HD>(row, chunk);
          next = CH / 2;
        } else {
          at = is_k ? kswz<HD>(row, chunk) : vseg<HD>(row, chunk);
        }
        *reinterpret_cast<u32x4*>(to + at * 8) = widen8<T>(u32x2{x[c][0], x[c][1]}, scale);
        *reinterpret_cast<u32x4*>(to + (at ^ next) * 8) = widen8<T>(u32x2{x[c][2], x[c][3]}, scale);
      }
    }
  };
  // The K tile staged with a V tile begins KLEAD keys later: the scores run that far ahead.
  constexpr int KLEAD = PIPE ? 32 : 0;
  auto issue_k = [&](const Places& p, int st) TT_INLINE {
    issue_half(true, p, sk + st * TILE, KLEAD / 16, k_bytes);
  };
  auto issue_v = [&](const Places& p, int st) TT_INLINE {
    issue_half(false, p, sv + st * TILE, 0, v_bytes);
  };
  // After the copies of this wave's V rows have landed: rows of keys behind the last that any row of the block sees are
  // cleared (0 times whatever lay there would not be 0), and where some rows of the block see keys that others do not,
  // infinities and NaN are taken out of V: 0 times those would reach the rows that do not see them.  Such values are
  // added to the rows that do see them at the end (restore_odd); `odd`: this wave took some out.
  const bool mixed = block_lo < block_end;
  bool odd = false;
  const auto odd_pair = [](uint32_t x) TT_INLINE -> uint32_t {  // of two values: bits 0 and 16
    constexpr uint32_t kCarry = (0x8000u - Num<T>::kExp) * 0x10001u;  // an exponent of ones carries into the sign
    return (((x & 0x7fff7fffu) + kCarry) >> 15) & 0x10001u;
  };
  auto settle_v = [&](int t0, int st) TT_INLINE {
    const int g0 = rw * WROWS;
    u32x4* const tile = reinterpret_cast<u32x4*>(sv + st * TILE + g0 * HD);
    const int n = min(max(kend - (t0 + g0), 0), WROWS);
    if (mixed && t0 + KT > block_lo) {
      for (int e = lane; e < n * CH; e += 64) {
        u32x4 x = tile[e];
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t m = odd_pair(x[i]);
          any |= m;
          x[i] &= ~(m * 0xffffu);
        }
        if (any != 0) {
          tile[e] = x;
          odd = true;
        }
      }
    }
    if (n < WROWS)
      for (int e = n * CH + lane; e < WROWS * CH; e += 64) tile[e] = u32x4{0u, 0u, 0u, 0u};
    lds_done();
  };
  // The same for the bytes of 16 keys of V from t0 on that a lane holds, with their scale: those that are no number in T.
  auto settle_bytes = [&](u32x2& x, int t0, uint32_t scale) TT_INLINE {
    const uint32_t carry = (0x80 - widen_limit<T>(scale)) * 0x01010101u;  // takes a byte that is none to 128 and above
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (mixed && t0 + 16 > block_lo) {
        const uint32_t m = (((x[i] & 0x7f7f7f7fu) + carry) >> 7) & 0x01010101u;
        odd |= m != 0;
        x[i] &= ~(m * 0xffu);
      }
      const int n = min(max(kend - (t0 + 8 * i + 4 * hf), 0), 4);  // keys before the end
      x[i] &= n == 4 ? ~0u : (1u << (8 * n)) - 1;
    }
  };
  auto land_v = [&](int t0, int st, const Scales& se, bool written = false) TT_INLINE {
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("" ::: "memory");
    if (C8 && PIPE && !written) {
      Bytes x;
      read_bytes(x, k_bytes);
      write_half(true, se, sk + st * TILE, KLEAD / 16, x);
      read_bytes(x, v_bytes);
      write_half(false, se, sv + st * TILE, 0, x);
      lds_done();
    }
    settle_v(t0, st);
    if constexpr (RW > 1) raw_barrier();
  };

  floatx16 o[DB];
  float m_ref, l_run, mc, thr;

  // Asked for after the first copies, which need addresses of their own first.  Branches are the wave's: where lanes went
  // around loads past head_dim by themselves, the compiler saved registers that every lane needs for the next tile in that
  // branch's last block, with half of the lanes off.
  v8 qf[KSTEPS];
  auto load_q = [&]() TT_INLINE {
    int width = hd;
    asm volatile("" : "+s"(width));  // (the comparisons would be kept in registers)
    const T* qp = static_cast<const T*>(a.q) + (int64_t)(sq.first + tok) * a.q_row + head * a.q_head;
    if constexpr (RAW) {  // features 32 j + 16 hf + {0..7} and the next 8, as a lane reads those of its keys
#pragma unroll
      for (int j = 0; j < KSTEPS / 2; ++j) {
        const u32x4 none = {0u, 0u, 0u, 0u};
        u32x4 x = none, y = none;
        if (32 * j + 16 < width) {
          x = *reinterpret_cast<const u32x4*>(qp + 32 * j + 16 * hf);
          y = *reinterpret_cast<const u32x4*>(qp + 32 * j + 16 * hf + 8);
        } else if (32 * j < width) {
          x = *reinterpret_cast<const u32x4*>(qp + 32 * j);
          y = *reinterpret_cast<const u32x4*>(qp + 32 * j + 8);
          x = hf == 0 ? x : none;
          y = hf == 0 ? y : none;
        }
        qf[2 * j] = __builtin_bit_cast(v8, x);
        qf[2 * j + 1] = __builtin_bit_cast(v8, y);
      }
    } else if (!FAR && width == HD) {
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk) qf[kk] = *reinterpret_cast<const v8*>(qp + 16 * kk + 8 * hf);
    } else {
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk) {
        const u32x4 none = {0u, 0u, 0u, 0u};
        u32x4 x = none;
        if (16 * kk + 8 < width) {
          x = *reinterpret_cast<const u32x4*>(qp + 16 * kk + 8 * hf);
        } else if (16 * kk < width) {
          x = *reinterpret_cast<const u32x4*>(qp + 16 * kk);
          x = hf == 0 ? x : none;
        }
        qf[kk] = __builtin_bit_cast(v8, x);
      }
    }
  };
  using Scores = floatx16;  // of 32 keys
  using Probs = v8[2];
  auto read_k = [&](int kk, int st, int kb) TT_INLINE -> v8 {  // 32 keys, features 16 kk + 8 hf + {0..7}
    const uint32_t stage = 2 * (st * TILE + kb * 32 * HD);
    const uint32_t at = FAR ? (kread[0] + stage) ^ (32 * kk) : kread[kk] + stage;
    return *(const __attribute__((address_space(3))) v8*)at;
  };
  auto read_v = [&](int i, int st, int kc) TT_INLINE -> v8 {
    // features 32 i + l % 32; keys 16 kc + 4 hf + {0..3} and 8 further: the order of the lane's probabilities
    const uint32_t stage = 2 * st * TILE, key = 2 * kc * 16 * HD;
    const uint32_t at = (FAR ? (vread[0] + stage) ^ (64 * i) : vread[i] + stage) + key;
    const shortx4 x0 = read_tr16((const lds_short*)at), x1 = read_tr16((const lds_short*)(at + 16 * HD));
    return __builtin_bit_cast(v8, shortx8{x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]});
  };
  // RAW: features 32 j + 16 hf + {0..15} of key l % 32; and features 32 i + l % 32 of the keys as above.
  auto read_kb = [&](int j, int st, int kb) TT_INLINE -> u32x4 {
    return *(const __attribute__((address_space(3))) u32x4*)(kread[j] + st * TILE + kb * 32 * ROW);
  };
  auto read_vb = [&](int i, int st, int kc) TT_INLINE -> u32x2 {
    return read_tr8((const lds_short*)(vread[i] + st * TILE + kc * 16 * ROW));
  };
  // FAR: one wave per SIMD, so nothing else runs while it waits for a fragment.  Fragments are read four products
  // before theirs (read just before, as registers are too few for the compiler to do otherwise by itself, prompts of
  // 4 x 4096 tokens on 16 heads of 256 took 1440 us; so 1120).
  constexpr int AHEAD = 4;
  auto ahead = [&](auto read, int reads, auto multiply, auto n) TT_INLINE {
    v8 x[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) x[j] = read(j);
    if (reads == 1) __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);  // LDS reads
    else __builtin_amdgcn_sched_group_barrier(0x100, 2 * AHEAD, 0);
#pragma unroll
    for (int j = 0; j < n; ++j) {
      multiply(j, x[j % AHEAD]);
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // a product
      if (j + AHEAD >= n) continue;
      x[j % AHEAD] = read(j + AHEAD);
      if (reads == 1) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      else __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
  };
  auto scores = [&](Scores& s, int st, int kb) TT_INLINE {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.f;
    if constexpr (FAR) {
      ahead([&](int kk) TT_INLINE { return read_k(kk, st, kb); }, 1,
            [&](int kk, v8 x) TT_INLINE { s = Num<T>::mfma(x, qf[kk], s); }, std::integral_constant<int, KSTEPS>{});
    } else {
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk) s = Num<T>::mfma(read_k(kk, st, kb), qf[kk], s);
    }
  };
  auto mask_scores = [&](Scores& s, int t0, uint32_t bad) TT_INLINE {
    if (t0 + 32 <= lim_lo && bad == 0) return;
    const int rem = lim - t0 - 4 * hf;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if ((bad >> (j >> 3)) & 1u) s[j] = __builtin_nanf("");
      s[j] = 8 * (j >> 2) + (j & 3) < rem ? s[j] : -INFINITY;
    }
  };
  auto row_max = [&](const Scores& s) TT_INLINE -> float {
    float mx = s[0];
#pragma unroll
    for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[j]);
    return xhalf_max(mx);
  };
  auto move_max = [&](float mt) TT_INLINE {
    if (__builtin_amdgcn_ballot_w64(mt > thr) == 0) return;
    const float m_new = fmaxf(m_ref, mt);
    const bool none = m_new == -INFINITY;  // no key of this row so far: o and l are 0
    const float corr = none ? 1.f : seq_weight((m_ref - m_new) * c2);
    m_ref = m_new;
    mc = none ? 0.f : m_new * c2 - Num<T>::kShift;
    thr = none ? -INFINITY : m_new + lazy;
    l_run *= corr;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] *= corr;
  };
  auto probabilities = [&](const Scores& s, Probs& p16) TT_INLINE {
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s[j], c2, -mc));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(s[j + 1], c2, -mc));
      p16[j >> 3][j & 7] = (T)p0;
      p16[j >> 3][(j & 7) + 1] = (T)p1;
    }
  };
  auto add_sums = [&](const Probs& p16) TT_INLINE {
#pragma unroll
    for (int j = 0; j < 16; j += 2) l_run = Num<T>::add2(v2{p16[j >> 3][j & 7], p16[j >> 3][(j & 7) + 1]}, l_run);
  };
  // The probabilities are made by here.
  auto pin = [&](Probs& p16) TT_INLINE {
#pragma unroll
    for (int c = 0; c < 2; ++c) asm volatile("" : "+v"(p16[c]));
  };
  auto add_values = [&](const Probs& p16, int st, int kb) TT_INLINE {
    if constexpr (FAR) {
      ahead([&](int j) TT_INLINE { return read_v(j % DB, st, 2 * kb + j / DB); }, 2,
            [&](int j, v8 x) TT_INLINE { o[j % DB] = Num<T>::mfma(x, p16[j / DB], o[j % DB]); },
            std::integral_constant<int, 2 * DB>{});
    } else {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < DB; ++i) o[i] = Num<T>::mfma(read_v(i, st, 2 * kb + c), p16[c], o[i]);
    }
  };
  {
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    m_ref = -INFINITY;  // the maximum that the sums are relative to, in units of the raw scores
    l_run = 0.f;        // this lane's half of the row's sum
    mc = 0.f;           // m_ref c log2(e) - kShift
    thr = -INFINITY;    // a tile maximum above this moves m_ref

    if constexpr (PIPE) {
      static_assert(KW == 1 && KT == 64, "two steps of 32 keys per tile");
      const int steps = wave_active && lim_hi > kbeg ? (lim_hi - kbeg + 31) / 32 : 0;  // of this wave
      int pe = 0, pe_next = 0;  // pages from this tile's and the next tile's first key on
      Scales se{0, 0};          // 8 bits: the scales there
      Scores sa, sb;
      float mt;
      char* const k_first = reinterpret_cast<char*>(sv + TILE) + rw * CPG * 1024;
      if (ntiles > 0) {
        if constexpr (PAGED) {
          pe = tile_pages(kbeg);
          pe_next = tile_pages(kbeg + KT);
        }
        const Places at = places(pe, kbeg);
        if constexpr (C8) se = tile_scales(pe, kbeg);
        // the first 32 keys go where the second half of a K tile before the first would lie
        // (8 bits: by way of the second V tile's place)
        issue_half(true, at, sk + TILE, -2, k_first);
        issue_k(at, 0);
        issue_v(at, 0);
      }
      load_q();
      if constexpr (C8) {
        __builtin_amdgcn_s_waitcnt(0);
        asm volatile("" ::: "memory");
        if (ntiles > 0) {
          Bytes x;
          read_bytes(x, k_first);
          write_half(true, se, sk + TILE, -2, x);
        }
      }
      land_v(kbeg, 0, se);
      if (steps > 0) {
        scores(sa, 1, 1);
        uint32_t bad = PAGED ? bad_groups(pe, kbeg) : 0;
        if constexpr (C8) bad |= bad_scales(se, kbeg);
        mask_scores(sa, kbeg, bad);
        mt = row_max(sa);
        move_max(mt);
      }
      lds_done();
      raw_barrier();  // the second tile's copies go where those first 32 keys lie
      // A step of 32 keys: the exps of its scores s run beside the products of the next 32 keys, and its P V beside
      // their maximum.
      auto step = [&](int t0, int st, int h, uint32_t bad, Scores& s, Scores& sn, bool widen = false) TT_INLINE {
        Probs p16;
        __builtin_amdgcn_sched_barrier(0);
        scores(sn, st, h);
        probabilities(s, p16);
        pin(p16);
        __builtin_amdgcn_sched_barrier(0);
        mask_scores(sn, t0 + 32 * (h + 1), bad >> (2 * h + 2));
        __builtin_amdgcn_s_setprio(1);  // (prompts take 1 to 3% longer without)
        Bytes kx, vx;  // of the next tile; what held the scores has room for them
        if (widen) {
          wait_vmcnt<0>();
          asm volatile("" ::: "memory");
          read_bytes(kx, k_bytes);
          read_bytes(vx, v_bytes);
        }
        add_sums(p16);
        add_values(p16, st, h);
        if (widen) {
          write_half(true, se, sk + (st ^ 1) * TILE, KLEAD / 16, kx);
          write_half(false, se, sv + (st ^ 1) * TILE, 0, vx);
        }
        mt = row_max(sn);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(0);
        move_max(mt);
      };
      auto last_step = [&](int st, int h, Scores& s) TT_INLINE {
        Probs p16;
        probabilities(s, p16);
        add_sums(p16);
        add_values(p16, st, h);
      };
      uint32_t bad = 0;
      // Packed keys: this wave's rows of the next tile, moved on by a tile at a time (working every tile's place out
      // from its number took the scalar unit some forty instructions more).
      const char *k_next = nullptr, *v_next = nullptr;
      if constexpr (!PAGED) {
        const int64_t row = sq.first + KT + rw * WROWS;
        k_next = reinterpret_cast<const char*>(kh) + 2 * (row + KLEAD) * a.k_row;
        v_next = reinterpret_cast<const char*>(vh) + 2 * row * a.v_row;
      }
      const auto bytes_of = [&](int left, int row) TT_INLINE -> uint32_t {  // of `left` rows, 16 at most
        const int n = min(left, 16);
        return n > 0 ? 2 * ((n - 1) * (uint32_t)row + hd) : 0;
      };
      auto fetch = [&](int r, int st) TT_INLINE {
        const int t0 = kbeg + r * KT;
        if constexpr (PAGED) bad = bad_groups(pe, t0);
        if constexpr (C8) bad |= bad_scales(se, t0);
        if (r + 1 >= ntiles) return;
        if constexpr (PAGED) {
          pe = pe_next;
          pe_next = tile_pages(t0 + 2 * KT);
          const Places at = places(pe, t0 + KT);
          if constexpr (C8) se = tile_scales(pe, t0 + KT);
          issue_k(at, st ^ 1);
          issue_v(at, st ^ 1);
        } else {
          static_assert(PG == 1, "16 rows of a tile per wave");
          const int left = keys - (t0 + KT + rw * WROWS);
          const __amdgpu_buffer_rsrc_t kr = buffer_rsrc(k_next, bytes_of(left - KLEAD, (int)a.k_row));
          const __amdgpu_buffer_rsrc_t vr = buffer_rsrc(v_next, bytes_of(left, (int)a.v_row));
          E* const kt = sk + (st ^ 1) * TILE + rw * WROWS * HD;
          E* const vt = sv + (st ^ 1) * TILE + rw * WROWS * HD;
#pragma unroll
          for (int c = 0; c < CPG; ++c) lds_copy16_buf(kr, koff[c], reinterpret_cast<half*>(kt + c * RPB * HD));
#pragma unroll
          for (int c = 0; c < CPG; ++c) lds_copy16_buf(vr, voff[c], reinterpret_cast<half*>(vt + c * RPB * HD));
          k_next += 2 * KT * a.k_row;
          v_next += 2 * KT * a.v_row;
        }
      };
      auto whole_tile = [&](int r, int st) TT_INLINE {
        const int t0 = kbeg + r * KT;
        fetch(r, st);
        step(t0, st, 0, bad, sa, sb);
        step(t0, st, 1, bad, sb, sa, BESIDE);
        land_v(t0 + KT, st ^ 1, se, BESIDE);
      };
      // Tiles both of whose steps have a next one, up to head_dim 128 two per pass so that their stages are constants
      // (beyond, the code would not fit the instruction cache); then this wave's last tile; then those that only
      // other waves of the block need.
      const int whole = max(steps - 1, 0) / 2;
      int r = 0;
      if constexpr (HD <= 128) {
        for (; r + 1 < whole; r += 2) {
          whole_tile(r, 0);
          whole_tile(r + 1, 1);
        }
        if (r < whole) whole_tile(r++, 0);
      } else {
        for (; r < whole; ++r) whole_tile(r, r & 1);
      }
      if (r < ntiles) {
        const int t0 = kbeg + r * KT;
        const int st = r & 1;
        fetch(r, st);
        if (steps - 2 * r == 2) {
          step(t0, st, 0, bad, sa, sb);
          last_step(st, 1, sb);
        } else if (steps - 2 * r == 1) {
          last_step(st, 0, sa);
        }
        for (++r; r < ntiles; ++r) {
          land_v(kbeg + r * KT, r & 1, se);
          fetch(r, r & 1);
        }
      }
    } else if constexpr (RAW) {
      // The same over an 8-bit cache, in tiles of KT keys: what a tile asks for besides its keys (pages, scales, masks,
      // waits) would take as long as 32 keys of half the bytes.  The scales of the tile after the next are asked for before
      // its copies, so that what waits for the copies has them too.
      static_assert(RW == 1, "a wave's own tiles");
      constexpr int COPIES = 2 * PG * CPG, KB = KT / 32;
      const int rounds = (ntiles - grp + KW - 1) / KW;
      const int t_first = kbeg + grp * KT;
      int pe0 = 0, pe1 = 0, pe2 = 0;
      Scales se0{0, 0}, se1{0, 0};
      if (rounds > 0) {
        pe0 = tile_pages(t_first);
        pe1 = tile_pages(t_first + KW * KT);
        pe2 = tile_pages(t_first + 2 * KW * KT);
        const Places at = places(pe0, t_first);
        se0 = tile_scales(pe0, t_first);
        se1 = tile_scales(pe1, t_first + KW * KT);
        load_q();
        issue_k(at, 0);
        issue_v(at, 0);
        if (rounds > 1) {
          const Places next = places(pe1, t_first + KW * KT);
          issue_k(next, 1);
          issue_v(next, 1);
          wait_vmcnt<(2 * COPIES < 63 ? 2 * COPIES : 63)>();
        } else {
          wait_vmcnt<COPIES>();
        }
        // (Q has come.  Left to itself, the compiler waits for it where it is used, in the loop, and there in every round for
        // all copies but the last two: 4 to 5% of 64 tokens over 8000 keys.)
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) asm volatile("" : "+v"(qf[kk]));
      }
      for (int r = 0; r < rounds; ++r) {
        const int t0 = t_first + r * KW * KT;
        const int st = r & 1;
        if (r + 1 < rounds) wait_vmcnt<COPIES>();
        else wait_vmcnt<0>();
        asm volatile("" ::: "memory");
        if constexpr (NH > 1) raw_barrier();  // every wave's copies have landed
        u32x4 kx[KB][KSTEPS / 2];
        u32x2 vx[2 * KB][DB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int j = 0; j < KSTEPS / 2; ++j) kx[kb][j] = read_kb(j, st, kb);
#pragma unroll
        for (int c = 0; c < 2 * KB; ++c)
#pragma unroll
          for (int i = 0; i < DB; ++i) vx[c][i] = read_vb(i, st, c);
        const uint32_t bad = bad_groups(pe0, t0) | bad_scales(se0, t0);
        const int pn = pe2;
        const Scales se = se0;
        pe0 = pe1;
        pe1 = pe2;
        pe2 = tile_pages(t0 + 3 * KW * KT);
        // (The empty asm moves the scales on here, and they are held as the bytes that they are loaded as: the compiler would
        // otherwise move or widen them at the end of the round, when the next ones are on their way, and wait for those, and
        // so for the copies behind them: 64 tokens over 8000 keys 196 -> 207 us.)
        uint32_t k1 = se1.k, v1 = se1.v;
        asm volatile("" : "+v"(k1), "+v"(v1));
        se0 = Scales{(uint8_t)k1, (uint8_t)v1};
        lds_done();
        if (r + 2 < rounds) {
          se1 = tile_scales(pn, t0 + 2 * KW * KT);
          if constexpr (NH > 1) raw_barrier();  // every wave has read this stage
          const Places at = places(pn, t0 + 2 * KW * KT);
          issue_k(at, st);
          issue_v(at, st);
        }
        if (t0 + KT > (mixed ? min(block_lo, kend) : kend)) {
#pragma unroll
          for (int c = 0; c < 2 * KB; ++c)
#pragma unroll
            for (int i = 0; i < DB; ++i) settle_bytes(vx[c][i], t0 + 16 * c, __builtin_amdgcn_readlane(se.v, c));
        }
        Scores s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const float k0 = scale_of(se, 2 * kb, true), k1 = scale_of(se, 2 * kb + 1, true), scale = col < 16 ? k0 : k1;
#pragma unroll
          for (int e = 0; e < 16; ++e) s[kb][e] = 0.f;
#pragma unroll
          for (int kk = 0; kk < KSTEPS; ++kk) {
            const u32x2 x = {kx[kb][kk / 2][2 * (kk & 1)], kx[kb][kk / 2][2 * (kk & 1) + 1]};
            s[kb] = Num<T>::mfma(__builtin_bit_cast(v8, widen8<T>(x, scale)), qf[kk], s[kb]);
          }
        }
        float scale_v[2 * KB];
#pragma unroll
        for (int c = 0; c < 2 * KB; ++c) scale_v[c] = scale_of(se, c, false);
        float mt = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          mask_scores(s[kb], t0 + 32 * kb, bad >> (2 * kb));
          mt = fmaxf(mt, row_max(s[kb]));
        }
        move_max(mt);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          Probs p16;
          probabilities(s[kb], p16);
          add_sums(p16);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < DB; ++i)
              o[i] = Num<T>::mfma(__builtin_bit_cast(v8, widen8<T>(vx[2 * kb + c][i], scale_v[2 * kb + c])), p16[c], o[i]);
        }
      }
    } else {
      // Tiles grp, grp + KW, ... by this wave alone.  The tile after the next is asked for as soon as this one's
      // fragments are in registers, so that close to two tiles are in flight all the time.
      static_assert(RW == 1 && KT == 32, "a wave's own tiles of 32 keys");
      constexpr int COPIES = 2 * PG * CPG;  // of a tile
      const int rounds = (ntiles - grp + KW - 1) / KW;
      const int t_first = kbeg + grp * KT;
      int pe0 = 0, pe1 = 0, pe2 = 0;  // pages of this tile, the next and the one after it
      if (rounds > 0) {
        if constexpr (PAGED) {
          pe0 = tile_pages(t_first);
          pe1 = tile_pages(t_first + KW * KT);
          pe2 = tile_pages(t_first + 2 * KW * KT);
        }
        const Places at = places(pe0, t_first);
        issue_k(at, 0);
        issue_v(at, 0);
        if (rounds > 1) {
          const Places next = places(pe1, t_first + KW * KT);
          issue_k(next, 1);
          issue_v(next, 1);
        }
      }
      load_q();
      for (int r = 0; r < rounds; ++r) {
        const int t0 = t_first + r * KW * KT;
        const int st = r & 1;
        // All but the next tile's copies, which were the last to be issued, have landed.
        if (r + 1 < rounds) wait_vmcnt<COPIES>();
        else wait_vmcnt<0>();
        asm volatile("" ::: "memory");
        settle_v(t0, st);
        // A wave has its SIMD to itself: all fragments are read before the first product, and only the first waits.
        v8 kf[KSTEPS], vf[2][DB];
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) kf[kk] = read_k(kk, st, 0);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < DB; ++i) vf[c][i] = read_v(i, st, c);
        __builtin_amdgcn_sched_barrier(0);
        Scores s;
        Probs p16;
        float mt;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) s = Num<T>::mfma(kf[kk], qf[kk], s);
        const uint32_t bad = PAGED ? bad_groups(pe0, t0) : 0;
        const int pn = pe2;
        if constexpr (PAGED) {
          pe0 = pe1;
          pe1 = pe2;
          pe2 = tile_pages(t0 + 3 * KW * KT);
        }
        if (r + 2 < rounds) {
          lds_done();
          const Places at = places(pn, t0 + 2 * KW * KT);
          issue_k(at, st);
          issue_v(at, st);
        }
        mask_scores(s, t0, bad);
        mt = row_max(s);
        move_max(mt);
        probabilities(s, p16);
        add_sums(p16);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < DB; ++i) o[i] = Num<T>::mfma(vf[c][i], p16[c], o[i]);
      }
    }
  }
  // Sums of this wave's rows over both halves of the wave.
  float l_row = xhalf_sum(l_run);

  // A sum that is NaN though its row's scores are not holds infinities of V (restore_odd); the sum of the sums tells, or
  // raises a false alarm.
  float all = 0.f;
#pragma unroll
  for (int i = 0; i < DB; ++i) {
    float sum = o[i][0];
#pragma unroll
    for (int e = 1; e < 16; ++e) sum += o[i][e];
    all += sum;
  }
  bool lost = all != all && l_row == l_row;
  if constexpr (C8 && RW > 1) {  // (the library's own would take LDS of its own, and the tiles and bytes fill it)
    if (mixed) {
      int* const flags = reinterpret_cast<int*>(seq_lds);
      __syncthreads();
      if (lane == 0) flags[wave] = 0;
      if (odd) flags[wave] = 1;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < RW; ++w) odd |= flags[w] != 0;
    }
  } else if (RW > 1 && mixed) {
    odd = __syncthreads_or(odd) != 0;
  }

  // Over the groups, by all of them: group g joins the g-th, (g + KW)-th, ... of the 4-feature pieces that a lane holds,
  // from [group][piece][lane] and (maximum, sum) in LDS.
  if constexpr (KW > 1) {
    static_assert(RW == 1, "groups are waves");
    floatx4* const pieces = reinterpret_cast<floatx4*>(seq_lds);
    float2* const sums = reinterpret_cast<float2*>(pieces + KW * DB * 4 * 64);
    int* const flags = reinterpret_cast<int*>(sums + KW * 32);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        pieces[(grp * DB * 4 + i * 4 + g) * 64 + lane] =
            floatx4{o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]};
    if (hf == 0) sums[grp * 32 + col] = make_float2(m_ref, l_row);
    const bool any_odd = __builtin_amdgcn_ballot_w64(odd) != 0, any_lost = __builtin_amdgcn_ballot_w64(lost) != 0;
    flags[grp] = (any_odd ? 1 : 0) | (any_lost ? 2 : 0);
    __syncthreads();
    int flag = 0;
#pragma unroll
    for (int g = 0; g < KW; ++g) flag |= flags[g];
    odd = (flag & 1) != 0, lost = (flag & 2) != 0;
    float2 ml[KW];
    float m = -INFINITY;
#pragma unroll
    for (int g = 0; g < KW; ++g) {
      ml[g] = sums[g * 32 + col];
      m = fmaxf(m, ml[g].x);
    }
    float w[KW], l = 0.f;
#pragma unroll
    for (int g = 0; g < KW; ++g) {
      // a group without a maximum saw no key (its sum, 0, is its weight) or only NaN (NaN is)
      w[g] = ml[g].x == -INFINITY ? ml[g].y : seq_weight((ml[g].x - m) * c2);
      l = fmaf(w[g], ml[g].y, l);
    }
    m_ref = m;
    l_row = l;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if ((i * 4 + g) % KW != grp) continue;
        floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KW; ++k) {
          const floatx4 y = pieces[(k * DB * 4 + i * 4 + g) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[e] = fmaf(w[k], y[e], sum[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][4 * g + e] = sum[e];
      }
  }

  // Whole rows of a wide block go out through LDS, 16 bytes per lane and rows side by side: straight from the
  // accumulators a store would touch 32 rows, 16 bytes of each.  (16-byte pieces are exchanged within their row by its
  // number, against bank conflicts.)
  if constexpr (RW > 1) {
    if (part < 0) {
      constexpr int SW = CH < 16 ? CH - 1 : 15;
      T* const tile = reinterpret_cast<T*>(seq_lds) + rw * 32 * HD;
      __syncthreads();
      const float inv = l_row == 0.f ? 0.f : 1.0f / l_row;  // no key: zeros
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          typedef T v4 __attribute__((ext_vector_type(4)));
          *reinterpret_cast<v4*>(tile + col * HD + (((4 * i + g) ^ (col & SW)) * 8 + 4 * hf)) =
              v4{(T)(o[i][4 * g] * inv), (T)(o[i][4 * g + 1] * inv), (T)(o[i][4 * g + 2] * inv),
                 (T)(o[i][4 * g + 3] * inv)};
        }
      lds_done();
      const int place = tok * a.heads + head;  // lane r holds row r's
      T* const out = static_cast<T*>(a.out) + (int64_t)sq.first * a.heads * hd;
#pragma unroll
      for (int e = 0; e < 32 * CH / 64; ++e) {
        const int r = e * RPC + lane / CH, c = lane % CH;
        const u32x4 x = *reinterpret_cast<const u32x4*>(tile + r * HD + ((c ^ (r & SW)) * 8));
        const int to = __shfl(place, r);
        if (wr0 + r < rows && 8 * c < hd) *reinterpret_cast<u32x4*>(out + (int64_t)to * hd + 8 * c) = x;
      }
    }
  }

  // Other output rows, or a part's sums: O and the sum in units of exp2(m - kShift), the maximum in log2 units.
  const int64_t part0 = ((int64_t)part * a.kv_heads + hkv) * R - r0;  // + row
  const int r = wr0 + col;
  if (r < rows) {
    if (part >= 0) {
      float* const dst = RW > 1 ? a.part_o + (part0 + r0) * hd + wide_place(hd, r - r0, 4 * hf)
                                : a.part_o + (part0 + r) * hd + 4 * hf;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (32 * i + 8 * g < hd && (i * 4 + g) % KW == grp)
            *reinterpret_cast<floatx4*>(dst + (4 * i + g) * (RW > 1 ? 256 : 8)) =
                floatx4{o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]};
      if (hf == 0 && grp == 0) a.part_ml[part0 + r] = make_float2(m_ref * c2, l_row);
    } else if constexpr (RW == 1) {
      const float inv = l_row == 0.f ? 0.f : 1.0f / l_row;
      T* dst = static_cast<T*>(a.out) + ((int64_t)(sq.first + tok) * a.heads + head) * hd;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (32 * i + 8 * g < hd && (i * 4 + g) % KW == grp) {
            typedef T v4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<v4*>(dst + 32 * i + 8 * g + 4 * hf) =
                v4{(T)(o[i][4 * g] * inv), (T)(o[i][4 * g + 1] * inv), (T)(o[i][4 * g + 2] * inv),
                   (T)(o[i][4 * g + 3] * inv)};
          }
    }
  }

  // restore_odd: the infinities and NaN of V.  No probability of a key that a row sees is 0 by the definition, so such a
  // value alone decides the sums that it enters.  Where settle_v took some out, or where a sum is NaN (an infinity times a
  // probability that is 0 in T), a wave adds them to what its rows that see them have in memory; adding one twice changes
  // nothing.  (A row with scores of -infinity only has no sum, and stays 0.)
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd || lost) != 0, 0)) {
    __builtin_amdgcn_s_waitcnt(0);
    __threadfence_block();
    if constexpr (KW > 1) __syncthreads();
    if (grp == 0 && wave_active) {
      int l = lane;
      asm volatile("" : "+v"(l));  // (what follows from it is worked out again instead of being held in registers)
      const int h = l >> 5, row = wr0 + (l & 31), r = min(row, rows - 1), token = r / G;
      const int seen = l_row == 0.f ? 0 : seq_limit(a, token, sq.count, keys);
      const bool any_lost = __builtin_amdgcn_ballot_w64(lost) != 0;
      T* const out =
          static_cast<T*>(a.out) + ((int64_t)(sq.first + token) * a.heads + hkv * G + r - token * G) * hd + 4 * h;
      float* const sum = RW > 1 ? a.part_o + (part0 + r0) * hd + wide_place(hd, r - r0, 4 * h)
                                : a.part_o + (part0 + r) * hd + 4 * h;
      typedef T v4 __attribute__((ext_vector_type(4)));
      const auto update = [&](int c, auto value) TT_INLINE {  // features 8 c + 4 h + {0..3} of this lane's row
        if (part >= 0) {
          floatx4* const dst = reinterpret_cast<floatx4*>(sum + c * (RW > 1 ? 256 : 8));
          floatx4 y = *dst;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = value(y[e], e);
          *dst = y;
        } else {
          v4* const dst = reinterpret_cast<v4*>(out + 8 * c);
          v4 y = *dst;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = (T)value((float)y[e], e);
          *dst = y;
        }
      };
      const auto values = [&](int key) TT_INLINE -> const Mem* {  // nullptr: in no page
        if constexpr (PAGED) {
          const int page = a.table[sq.seq * a.table_row + (key >> a.page_shift)];
          if ((uint32_t)page >= (uint32_t)a.pages) return nullptr;
          return vh + hw * a.v_head + page * a.v_page + (key & ((1 << a.page_shift) - 1)) * a.v_row;
        } else {
          return vh + (int64_t)(sq.first + key) * a.v_row;
        }
      };
      if (any_lost && row < rows && l_row == l_row)
        for (int c = 0; 8 * c < hd; ++c) update(c, [](float y, int) TT_INLINE { return y != y ? 0.f : y; });
      // 8 bits: the scale of a key's V (a key without one is NaN in all rows that see it, as its scores are)
      const auto scale_at = [&](int key) TT_INLINE -> float {
        const int page = a.table[sq.seq * a.table_row + (key >> a.page_shift)];
        const int block = (key & ((1 << a.page_shift) - 1)) >> a.block_shift;
        const uint32_t e = a.v_scale[page * a.s_page + block * a.s_block + hkv * a.s_head];
        return e8m0(e == 255 ? 0 : e);
      };
      for (int k0 = any_lost ? kbeg : kbeg + max(block_lo - kbeg, 0) / KT * KT; k0 < lim_hi; k0 += RPC) {
        const int key = min(k0 + l / CH, lim_hi - 1);
        const Mem* const vp = values(key);  // RPC keys, 8 values per lane
        u32x4 x = {0u, 0u, 0u, 0u};
        if (vp != nullptr && l % CH * 8 < hd) {
          if constexpr (C8) x = widen8<T>(*reinterpret_cast<const u32x2*>(vp + l % CH * 8), scale_at(key));
          else x = *reinterpret_cast<const u32x4*>(vp + l % CH * 8);
        }
        uint64_t found =
            __builtin_amdgcn_ballot_w64((odd_pair(x[0]) | odd_pair(x[1]) | odd_pair(x[2]) | odd_pair(x[3])) != 0);
        for (; found != 0; found &= found - 1) {
          const int n = __ffsll((unsigned long long)found) - 1, c = n % CH, key = min(k0 + n / CH, lim_hi - 1);
          v4 z;
          if constexpr (C8) {
            const u32x4 y = widen8<T>(*reinterpret_cast<const u32x2*>(values(key) + 8 * c), scale_at(key));
            z = __builtin_bit_cast(v4, h == 0 ? u32x2{y[0], y[1]} : u32x2{y[2], y[3]});
          } else {
            z = *reinterpret_cast<const v4*>(values(key) + 8 * c + 4 * h);
          }
          if (row < rows && key < seen)
            update(c, [&](float y, int e) TT_INLINE {
              const T w = z[e];
              return (__builtin_bit_cast(uint16_t, w) & Num<T>::kExp) == Num<T>::kExp ? y + (float)w : y;
            });
        }
      }
    }
  }
  if (!shares || x >= share_end) return;
  __syncthreads();  // the next tile's copies go where this one's may still be read
  }
}

}  // namespace tt
