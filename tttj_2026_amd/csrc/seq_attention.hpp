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
// A block owns 32 RW rows of one (sequence, kv head) and a range of keys.  Its waves form KW groups of RW: the waves
// of a group share key tiles of KT keys, staged in LDS two deep, and each owns 32 rows; the groups take alternate
// tiles and are merged through LDS at the end.  RW 4, KW 1 is the tile for many rows (bound by the matrix unit and
// exp), RW 1 with KW 2 or 4 the one for single tokens (bound by HBM: every wave streams tiles of its own, without a
// barrier).  Keys are also split over blocks where rows are few; seq_merge_kernel joins those parts.
//
// Per wave and tile: S^T = K Q^T with v_mfma_f32_32x32x16 (lane l holds row l % 32; of its 32 keys per block those
// with bit 2 equal to l / 32), softmax with a running maximum and sum in fp32, O^T += V^T P^T.  K and V stay in the
// row-major form of the projections and of the cache: ds_read_b64_tr_b16 transposes V on its way from LDS, and reads
// the keys in the order in which a lane holds its probabilities, so neither needs a shuffle.
// Scores are multiplied by c log2(e) in fp32 (rounding q c to 16 bits would cost as much precision as rounding the
// probabilities does).  Probabilities are rounded to the type of V for the matrix unit, relative to a maximum that
// is moved only when it grows by more than 2^8 (lazy rescaling), and times 2^7, so that fp16 holds what is down to
// 2^-31 of the largest: 100000 keys of 2^-25 each still count.
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
  static __device__ __forceinline__ floatx16 mfma(v8 a, v8 b, floatx16 c) { return mfma32x32x16(a, b, c); }
  static __device__ __forceinline__ float add2(v2 p, float c) {
    return __builtin_amdgcn_fdot2(p, v2{(half)1.f, (half)1.f}, c, false);
  }
};
template <>
struct Num<bf16> {
  using v2 = bf16x2;
  using v8 = bf16x8;
  static constexpr uint16_t kExp = 0x7f80;
  static __device__ __forceinline__ floatx16 mfma(v8 a, v8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(v2 p, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(p, v2{(bf16)1.f, (bf16)1.f}, c, false);
  }
};

// ds_read_b64_tr_b16 (16 lanes transpose their 4 rows of 16).  The __restrict gives the read alias information;
// without any, the compiler lets it wait for every global -> LDS copy in flight.
using lds_short = __attribute__((address_space(3))) short;
__device__ __forceinline__ shortx4 read_tr16(const lds_short* __restrict__ p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4*)p);
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const lds_short*)p;
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
  int slots;               // row tiles of the launch per kv head
  int splits, chunk;       // key ranges of `chunk` keys, `splits` of them at most
  float* part_o;           // [splits][tokens * heads][head_dim] where splits > 1
  float2* part_ml;         // [splits][tokens * heads]: maximum (log2 domain) and sum
};

constexpr float kSeqLazy = 8.0f;   // log2 growth of a row's maximum that moves its reference
constexpr float kSeqShift = 7.0f;  // log2 of the factor on the probabilities: 2^(8 + 7) < 65504

// V tiles are read by ds_read_b64_tr_b16: half a wave reads 64 bytes of each of 4 consecutive rows.  The 64-byte
// segments of a row are exchanged by its number so that those 4 pieces lie in different quarters of the 64 banks.
template <int HD>
__device__ __forceinline__ int vseg(int row, int c) {
  if constexpr (HD >= 128) return c ^ ((row & 3) << 2);
  else if constexpr (HD == 64) return c ^ ((row & 2) << 1);
  else return c;
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

template <typename T, int HD, int CB, int RW, int KW, int KT, bool PAGED, int WPE = (HD <= 64 ? 3 : HD <= 128 ? 2 : 1)>
__global__ __launch_bounds__(64 * RW * KW) __attribute__((amdgpu_waves_per_eu(WPE, WPE))) void seq_attention_kernel(SeqAttnArgs a) {
  using v2 = typename Num<T>::v2;
  using v8 = typename Num<T>::v8;
  constexpr int WR = 32 * CB;               // rows of a wave
  constexpr int R = WR * RW;
  constexpr bool PIPE = RW > 1;              // softmax beside the next keys' products
  constexpr int SB = PIPE ? 1 : KT / 32;    // 32-key blocks whose scores are taken at once
  constexpr int KSTEPS = HD / 16;           // k-steps of S^T
  constexpr int DB = HD / 32;               // 32-row blocks of O^T
  constexpr int CH = HD / 8;                // 16-byte chunks of a row
  constexpr int RPC = 64 / CH;              // rows per 1 KiB copy
  constexpr int WROWS = KT / RW;            // rows of a tile that one wave copies
  constexpr int PG = WROWS / 16;            // ... in groups of 16, each of which lies in one page
  constexpr int CPG = 16 / RPC;             // copies per group
  constexpr int TILE = KT * HD;
  static_assert(WROWS % 16 == 0 && RPC <= 16, "a wave copies whole 16-row groups");

  extern __shared__ __align__(16) char seq_lds[];

  const int hkv = blockIdx.x % a.kv_heads;
  const int rest = blockIdx.x / a.kv_heads;
  const int split = rest / a.slots;
  int slot = rest - split * a.slots;
  if (a.causal) slot = a.slots - 1 - slot;  // the heaviest tiles of a sequence first
  const SeqTile sq = seq_tile(a, slot, R);
  const int G = a.group;
  const int rows = sq.count * G;
  const int r0 = sq.tile * R;
  if (sq.tile < 0 || r0 >= rows) return;
  const int keys = seq_keys<PAGED>(a, sq.seq, sq.count);
  const int kbeg = split * a.chunk;
  const int block_end = seq_limit(a, min(r0 + R - 1, rows - 1) / G, sq.count, keys);
  if (split > 0 && kbeg >= block_end) return;
  // the last range takes what is left, should a sequence be longer than the launch was sized for
  const int kend = split == a.splits - 1 ? block_end : min(block_end, kbeg + a.chunk);
  const int ntiles = (kend - kbeg + KT - 1) / KT;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = RW == 1 ? 0 : wave % RW, grp = RW == 1 ? wave : wave / RW;
  const int hf = lane >> 5, col = lane & 31;
  T* const sk = reinterpret_cast<T*>(seq_lds) + (size_t)grp * 2 * TILE;
  T* const sv = reinterpret_cast<T*>(seq_lds) + (size_t)KW * 2 * TILE + (size_t)grp * 2 * TILE;

  // Rows of this wave; those behind the last repeat it and are not stored, so limits rise along the rows.
  const int wr0 = r0 + rw * WR;
  const bool wave_active = wr0 < rows;
  const int block_lo = seq_limit(a, r0 / G, sq.count, keys);  // the first row's
  const int lim_lo = seq_limit(a, min(wr0, rows - 1) / G, sq.count, keys);
  const int lim_hi = min(seq_limit(a, min(wr0 + WR - 1, rows - 1) / G, sq.count, keys), kend);
  int tok[CB], head[CB], lim[CB];
#pragma unroll
  for (int b = 0; b < CB; ++b) {
    const int r = min(wr0 + 32 * b + col, rows - 1);
    tok[b] = r / G;
    head[b] = hkv * G + r - tok[b] * G;
    lim[b] = seq_limit(a, tok[b], sq.count, keys);
  }

  // Copy sources: lane l of copy c of a group fetches row c RPC + l / CH of the group into the next 16 bytes of
  // LDS, from the chunk that belongs there.  Chunks at or past head_dim lie outside the buffer: LDS keeps the zeros
  // that it is cleared to (or receives those that such a load returns).
  const int hd = a.head_dim;
  uint32_t koff[CPG], voff[CPG];
#pragma unroll
  for (int c = 0; c < CPG; ++c) {
    const int row = c * RPC + lane / CH;
    const int kc = kswz<HD>(row, lane % CH) * 8, vc = vseg<HD>(row, lane % CH) * 8;
    koff[c] = kc < hd ? (uint32_t)(row * (int)a.k_row + kc) * 2 : 0x80000000u;
    voff[c] = vc < hd ? (uint32_t)(row * (int)a.v_row + vc) * 2 : 0x80000000u;
  }
  const T* const kh = static_cast<const T*>(a.k) + hkv * a.k_head;
  const T* const vh = static_cast<const T*>(a.v) + hkv * a.v_head;

  // Paged: lane l holds the page of the 16-key group l behind key t0 (of the first 8).
  auto tile_pages = [&](int t0) TT_INLINE -> int {
    const int key = min(t0 + 16 * (lane & 7), max(keys - 1, 0));
    return a.table[sq.seq * a.table_row + (key >> a.page_shift)];
  };
  // Which of those lie outside the cache (a bit each); their keys are not read and count as NaN.
  auto bad_groups = [&](int pe, int t0) TT_INLINE -> uint32_t {
    return (uint32_t)__ballot((uint32_t)pe >= (uint32_t)a.pages && t0 + 16 * lane < keys) & 0xffu;
  };
  auto issue_half = [&](const T* h, int64_t page_stride, int64_t row_stride, const uint32_t (&off)[CPG], T* tile, int t0,
                        int pe, int pe_lane) TT_INLINE {
#pragma unroll
    for (int p = 0; p < PG; ++p) {
      const int g0 = rw * WROWS + p * 16;
      const int t = t0 + g0;
      const int n = t < kbeg ? 0 : min(max(keys - t, 0), 16);
      const T* src;
      if constexpr (PAGED) {
        const int e = __builtin_amdgcn_readlane(pe, max(pe_lane + g0 / 16, 0));
        const int page = (uint32_t)e < (uint32_t)a.pages ? e : 0;
        src = h + page * page_stride + (t & ((1 << a.page_shift) - 1)) * row_stride;
      } else {
        src = h + (int64_t)(sq.first + max(min(t, keys - 1), 0)) * row_stride;
      }
      const __amdgpu_buffer_rsrc_t r = buffer_rsrc(src, n == 0 ? 0 : (uint32_t)((n - 1) * (int)row_stride + hd) * 2);
#pragma unroll
      for (int c = 0; c < CPG; ++c)
        lds_copy16_buf(r, off[c], reinterpret_cast<half*>(tile + (g0 + c * RPC) * HD));
    }
  };
  // The K tile staged with a V tile from key t0 begins KLEAD keys later: the scores run that far ahead.
  constexpr int KLEAD = PIPE ? 32 : 0;
  auto issue_k = [&](int t0, int st, int pe) TT_INLINE {
    issue_half(kh, a.k_page, a.k_row, koff, sk + st * TILE, t0 + KLEAD, pe, KLEAD / 16);
  };
  auto issue_v = [&](int t0, int st, int pe) TT_INLINE {
    issue_half(vh, a.v_page, a.v_row, voff, sv + st * TILE, t0, pe, 0);
  };
  // This wave's copies have landed, and the waves of the block meet.  Before that, V rows of keys behind the last are
  // cleared (0 times whatever lay there would not be 0), and where some rows of the block see keys that others do
  // not, infinities and NaN are taken out of V: 0 times those would reach the rows that do not see them.  Such values
  // are added to the rows that do see them at the end (restore_odd).
  const bool mixed = block_lo < block_end;
  bool odd = false;
  auto land_v = [&](int t0, int st) TT_INLINE {
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("" ::: "memory");
    const int g0 = rw * WROWS;
    u32x4* const tile = reinterpret_cast<u32x4*>(sv + st * TILE + g0 * HD);
    const int n = min(max(keys - (t0 + g0), 0), WROWS);
    if (mixed && t0 + KT > block_lo) {
      constexpr uint32_t kCarry = (0x8000u - Num<T>::kExp) * 0x10001u;  // an exponent of ones carries into the sign
      for (int e = lane; e < n * CH; e += 64) {
        u32x4 x = tile[e];
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t m = (((x[i] & 0x7fff7fffu) + kCarry) >> 15) & 0x10001u;
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
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
    if constexpr (RW > 1) raw_barrier();
  };

  if (hd < HD) {
    for (int e = tid; e < 4 * KW * TILE / 8; e += 64 * RW * KW)
      reinterpret_cast<u32x4*>(seq_lds)[e] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
  }

  v8 qf[CB][KSTEPS];
#pragma unroll
  for (int b = 0; b < CB; ++b) {
    const T* qp = static_cast<const T*>(a.q) + (int64_t)(sq.first + tok[b]) * a.q_row + head[b] * a.q_head;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      if (16 * kk + 8 * hf < hd) qf[b][kk] = *reinterpret_cast<const v8*>(qp + 16 * kk + 8 * hf);
      else qf[b][kk] = __builtin_bit_cast(v8, u32x4{0u, 0u, 0u, 0u});
    }
  }

  const float c2 = a.scale_log2, lazy = kSeqLazy / a.scale_log2;
  // LDS addresses of this lane's pieces of the first K and V block of a stage; the others lie at constant distances.
  // (The empty asm keeps each in one register: the compiler would spread the sums over many.)
  uint32_t kread[KSTEPS], vread[DB];
#pragma unroll
  for (int kk = 0; kk < KSTEPS; ++kk) {
    kread[kk] = lds_address(sk + col * HD + kswz<HD>(col, 2 * kk + hf) * 8);
    asm volatile("" : "+v"(kread[kk]));
  }
  const int vrow = 4 * hf + ((lane >> 2) & 3);
#pragma unroll
  for (int i = 0; i < DB; ++i) {
    const int c = vseg<HD>(vrow, 4 * i + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1));
    vread[i] = lds_address(sv + vrow * HD + c * 8 + 4 * (lane & 1));
    asm volatile("" : "+v"(vread[i]));
  }
  floatx16 o[CB][DB];
  float m_ref[CB], l_run[CB], mc[CB], thr[CB];

  using Scores = floatx16[CB][SB];
  using Probs = v8[CB][SB][2];
  auto scores = [&](Scores& s, int st, int kb0) TT_INLINE {
#pragma unroll
    for (int kb = 0; kb < SB; ++kb)
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk) {
        const v8 x = *(const __attribute__((address_space(3))) v8*)(kread[kk] + 2 * (st * TILE + (kb0 + kb) * 32 * HD));
#pragma unroll
        for (int b = 0; b < CB; ++b) {
          if (kk == 0) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[b][kb][e] = 0.f;
          }
          s[b][kb] = Num<T>::mfma(x, qf[b][kk], s[b][kb]);
        }
      }
  };
  auto mask_scores = [&](Scores& s, int t0, uint32_t bad) TT_INLINE {
    if (t0 + 32 * SB <= lim_lo && bad == 0) return;
#pragma unroll
    for (int b = 0; b < CB; ++b) {
      const int rem = lim[b] - t0 - 4 * hf;
#pragma unroll
      for (int kb = 0; kb < SB; ++kb)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if ((bad >> (2 * kb + (j >> 3))) & 1u) s[b][kb][j] = __builtin_nanf("");
          s[b][kb][j] = 32 * kb + 8 * (j >> 2) + (j & 3) < rem ? s[b][kb][j] : -INFINITY;
        }
    }
  };
  auto row_max = [&](const Scores& s, float (&mt)[CB]) TT_INLINE {
#pragma unroll
    for (int b = 0; b < CB; ++b) {
      float mx = s[b][0][0];
#pragma unroll
      for (int kb = 0; kb < SB; ++kb)
#pragma unroll
        for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[b][kb][j]);
      mt[b] = xhalf_max(mx);
    }
  };
  auto move_max = [&](const float (&mt)[CB]) TT_INLINE {
    bool grows = mt[0] > thr[0];
#pragma unroll
    for (int b = 1; b < CB; ++b) grows |= mt[b] > thr[b];
    if (__builtin_amdgcn_ballot_w64(grows) == 0) return;
#pragma unroll
    for (int b = 0; b < CB; ++b) {
      const float m_new = fmaxf(m_ref[b], mt[b]);
      const bool none = m_new == -INFINITY;  // no key of this row so far: o and l are 0
      const float corr = none ? 1.f : __builtin_amdgcn_exp2f((m_ref[b] - m_new) * c2);
      m_ref[b] = m_new;
      mc[b] = none ? 0.f : m_new * c2 - kSeqShift;
      thr[b] = none ? -INFINITY : m_new + lazy;
      l_run[b] *= corr;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[b][i][e] *= corr;
    }
  };
  auto probabilities = [&](const Scores& s, Probs& p16) TT_INLINE {
#pragma unroll
    for (int b = 0; b < CB; ++b)
#pragma unroll
      for (int kb = 0; kb < SB; ++kb)
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(s[b][kb][j], c2, -mc[b]));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(s[b][kb][j + 1], c2, -mc[b]));
          p16[b][kb][j >> 3][j & 7] = (T)p0;
          p16[b][kb][j >> 3][(j & 7) + 1] = (T)p1;
        }
  };
  auto add_sums = [&](const Probs& p16) TT_INLINE {
#pragma unroll
    for (int b = 0; b < CB; ++b)
#pragma unroll
      for (int kb = 0; kb < SB; ++kb)
#pragma unroll
        for (int j = 0; j < 16; j += 2)
          l_run[b] = Num<T>::add2(v2{p16[b][kb][j >> 3][j & 7], p16[b][kb][j >> 3][(j & 7) + 1]}, l_run[b]);
  };
  // The probabilities are made by here.
  auto pin = [&](Probs& p16) TT_INLINE {
#pragma unroll
    for (int b = 0; b < CB; ++b)
#pragma unroll
      for (int kb = 0; kb < SB; ++kb)
#pragma unroll
        for (int c = 0; c < 2; ++c) asm volatile("" : "+v"(p16[b][kb][c]));
  };
  auto add_values = [&](const Probs& p16, int st, int kb0) TT_INLINE {
#pragma unroll
    for (int kb = 0; kb < SB; ++kb)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < DB; ++i) {
          // keys 32 kb + 16 c + 4 hf + {0..3} and 8 further: the order of the lane's probabilities
          const uint32_t at = vread[i] + 2 * (st * TILE + (32 * (kb0 + kb) + 16 * c) * HD);
          const shortx4 x0 = read_tr16((const lds_short*)at);
          const shortx4 x1 = read_tr16((const lds_short*)(at + 16 * HD));
          const shortx8 x = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
#pragma unroll
          for (int b = 0; b < CB; ++b) o[b][i] = Num<T>::mfma(__builtin_bit_cast(v8, x), p16[b][kb][c], o[b][i]);
        }
  };
  {
#pragma unroll
    for (int b = 0; b < CB; ++b) {
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[b][i][e] = 0.f;
      m_ref[b] = -INFINITY;  // the maximum that the sums are relative to, in units of the raw scores
      l_run[b] = 0.f;        // this lane's half of the row's sum
      mc[b] = 0.f;           // m_ref c log2(e) - 7
      thr[b] = -INFINITY;    // a tile maximum above this moves m_ref
    }

    // Tiles of this wave's group, and those of them that its rows see.
    [[maybe_unused]] const int rounds = RW == 1 ? (ntiles - grp + KW - 1) / KW : (ntiles + KW - 1) / KW;
    const int tiles_w = wave_active && lim_hi > kbeg ? (lim_hi - kbeg + KT - 1) / KT : 0;
    [[maybe_unused]] const int rounds_w = (tiles_w - grp + KW - 1) / KW;
    [[maybe_unused]] const int t_first = kbeg + grp * KT;  // first key of the group's first tile
    if constexpr (PIPE) {
      static_assert(KW == 1 && KT == 64, "two steps of 32 keys per tile");
      const int steps = wave_active && lim_hi > kbeg ? (lim_hi - kbeg + 31) / 32 : 0;  // of this wave
      int pe = 0, pe_next = 0;  // pages from this tile's and the next tile's first key on
      Scores sa, sb;
      float mt[CB];
      if (ntiles > 0) {
        if constexpr (PAGED) {
          pe = tile_pages(kbeg);
          pe_next = tile_pages(kbeg + KT);
        }
        // the first 32 keys go where the second half of a K tile before the first would lie
        issue_half(kh, a.k_page, a.k_row, koff, sk + TILE, kbeg - 32, pe, -2);
        issue_k(kbeg, 0, pe);
        issue_v(kbeg, 0, pe);
      }
      land_v(kbeg, 0);
      if (steps > 0) {
        scores(sa, 1, 1);
        mask_scores(sa, kbeg, PAGED ? bad_groups(pe, kbeg) : 0);
        row_max(sa, mt);
        move_max(mt);
      }
      // A step of 32 keys: the exps of its scores s run beside the products of the next 32 keys, and its P V beside
      // their maximum.
      auto step = [&](int t0, int st, int h, uint32_t bad, Scores& s, Scores& sn) TT_INLINE {
        Probs p16;
        __builtin_amdgcn_sched_barrier(0);
        scores(sn, st, h);
        probabilities(s, p16);
        pin(p16);
        __builtin_amdgcn_sched_barrier(0);
        mask_scores(sn, t0 + 32 * (h + 1), bad >> (2 * h + 2));
        __builtin_amdgcn_s_setprio(1);
        add_sums(p16);
        add_values(p16, st, h);
        row_max(sn, mt);
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
      auto fetch = [&](int r, int st) TT_INLINE {
        const int t0 = kbeg + r * KT;
        if constexpr (PAGED) bad = bad_groups(pe, t0);
        if (r + 1 >= ntiles) return;
        pe = pe_next;
        if constexpr (PAGED) pe_next = tile_pages(t0 + 2 * KT);
        issue_k(t0 + KT, st ^ 1, pe);
        issue_v(t0 + KT, st ^ 1, pe);
      };
      auto whole_tile = [&](int r, int st) TT_INLINE {
        const int t0 = kbeg + r * KT;
        fetch(r, st);
        step(t0, st, 0, bad, sa, sb);
        step(t0, st, 1, bad, sb, sa);
        land_v(t0 + KT, st ^ 1);
      };
      // Tiles both of whose steps have a next one, two per pass so that their stages are constants; then this wave's
      // last tile; then those that only other waves of the block need.
      const int whole = max(steps - 1, 0) / 2;
      int r = 0;
      for (; r + 1 < whole; r += 2) {
        whole_tile(r, 0);
        whole_tile(r + 1, 1);
      }
      if (r < whole) whole_tile(r++, 0);
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
          land_v(kbeg + r * KT, r & 1);
          fetch(r, r & 1);
        }
      }
    } else {
      int pe = 0, pe_next = 0;
      if (grp < ntiles) {
        if constexpr (PAGED) {
          pe = tile_pages(t_first);
          pe_next = tile_pages(t_first + KW * KT);
        }
        issue_k(t_first, 0, pe);
        issue_v(t_first, 0, pe);
      }
      land_v(t_first, 0);
      for (int r = 0; r < rounds; ++r) {
        const int t = r * KW + grp;
        const int t0 = kbeg + t * KT;
        const int st = r & 1;
        const uint32_t bad = PAGED ? bad_groups(pe, t0) : 0;
        if (t + KW < ntiles) {
          pe = pe_next;
          if constexpr (PAGED) pe_next = tile_pages(t0 + 2 * KW * KT);
          issue_k(t0 + KW * KT, st ^ 1, pe);
          issue_v(t0 + KW * KT, st ^ 1, pe);
        }
        if (r < rounds_w) {
          Scores s;
          Probs p16;
          float mt[CB];
          scores(s, st, 0);
          mask_scores(s, t0, bad);
          row_max(s, mt);
          move_max(mt);
          probabilities(s, p16);
          add_sums(p16);
          add_values(p16, st, 0);
        }
        if (r + 1 < rounds) land_v(t0 + KW * KT, st ^ 1);
      }
    }
  }
  if (RW * KW > 1 && mixed) odd = __syncthreads_or(odd);

  if constexpr (KW > 1) {
    static_assert(CB == 1, "groups of waves hold one block of rows");
    // [group - 1][wave of the group][value][lane]: O, the maximum in log2 units and this lane's half of the sum
    constexpr int NV = DB * 16 + 2;
    float* const mrg = reinterpret_cast<float*>(seq_lds);
    __syncthreads();
    if (grp > 0) {
      float* p = mrg + (size_t)((grp - 1) * RW + rw) * NV * 64 + lane;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) p[(i * 16 + e) * 64] = o[0][i][e];
      p[(NV - 2) * 64] = m_ref[0];
      p[(NV - 1) * 64] = l_run[0];
    }
    __syncthreads();
    if (grp > 0) return;
#pragma unroll 1
    for (int g = 0; g < KW - 1; ++g) {
      const float* p = mrg + (size_t)(g * RW + rw) * NV * 64 + lane;
      const float m_g = p[(NV - 2) * 64], l_g = p[(NV - 1) * 64];
      const float m_new = fmaxf(m_ref[0], m_g);
      // a part without a maximum saw no key (its sum, 0, is then its weight) or only NaN (NaN is)
      const float c0 = m_ref[0] == -INFINITY ? l_run[0] : __builtin_amdgcn_exp2f((m_ref[0] - m_new) * c2);
      const float c1 = m_g == -INFINITY ? l_g : __builtin_amdgcn_exp2f((m_g - m_new) * c2);
      l_run[0] = l_run[0] * c0 + l_g * c1;
      m_ref[0] = m_new;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[0][i][e] = o[0][i][e] * c0 + p[(i * 16 + e) * 64] * c1;
    }
  }

#pragma unroll
  for (int b = 0; b < CB; ++b) {
    const float l = xhalf_sum(l_run[b]);
    if (wr0 + 32 * b + col >= rows) continue;
    const int64_t orow = (int64_t)(sq.first + tok[b]) * a.heads + head[b];
    if (lim[b] > a.chunk) {  // this row's keys lie in several parts
      float* dst = a.part_o + ((int64_t)split * a.tokens * a.heads + orow) * hd;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (32 * i + 8 * g < hd)
            *reinterpret_cast<floatx4*>(dst + 32 * i + 8 * g + 4 * hf) =
                floatx4{o[b][i][4 * g], o[b][i][4 * g + 1], o[b][i][4 * g + 2], o[b][i][4 * g + 3]};
      if (hf == 0) a.part_ml[(int64_t)split * a.tokens * a.heads + orow] = make_float2(m_ref[b] * c2, l);
      continue;
    }
    if (split > 0) continue;
    const float inv = l == 0.f ? 0.f : 1.0f / l;  // no key: zeros
    T* dst = static_cast<T*>(a.out) + orow * hd;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (32 * i + 8 * g < hd) {
          typedef T v4 __attribute__((ext_vector_type(4)));
          *reinterpret_cast<v4*>(dst + 32 * i + 8 * g + 4 * hf) =
              v4{(T)(o[b][i][4 * g] * inv), (T)(o[b][i][4 * g + 1] * inv), (T)(o[b][i][4 * g + 2] * inv),
                 (T)(o[b][i][4 * g + 3] * inv)};
        }
  }

  if (!mixed || __builtin_amdgcn_ballot_w64(odd) == 0) return;
  // restore_odd: a wave adds the infinities and NaN of V that were taken out to those of its rows that see them.
  __threadfence_block();
  const int from = kbeg + max(block_lo - kbeg, 0) / KT * KT;
  for (int key = from; key < lim_hi; ++key) {
    const T* vp = vh;
    if constexpr (PAGED) {
      const int page = a.table[sq.seq * a.table_row + (key >> a.page_shift)];
      if ((uint32_t)page >= (uint32_t)a.pages) continue;
      vp += page * a.v_page + (key & ((1 << a.page_shift) - 1)) * a.v_row;
    } else {
      vp += (int64_t)(sq.first + key) * a.v_row;
    }
    for (int d = lane; d < hd; d += 64) {
      const T x = vp[d];
      if ((__builtin_bit_cast(uint16_t, x) & Num<T>::kExp) != Num<T>::kExp) continue;
      for (int r = wr0; r < min(wr0 + WR, rows); ++r) {
        const int token = r / G, seen = seq_limit(a, token, sq.count, keys);
        if (key >= seen || (split > 0 && seen <= a.chunk)) continue;
        const int64_t orow = (int64_t)(sq.first + token) * a.heads + hkv * G + r - token * G;
        if (seen > a.chunk) a.part_o[((int64_t)split * a.tokens * a.heads + orow) * hd + d] += (float)x;
        else static_cast<T*>(a.out)[orow * hd + d] = (T)((float)static_cast<T*>(a.out)[orow * hd + d] + (float)x);
      }
    }
  }
}

}  // namespace tt
