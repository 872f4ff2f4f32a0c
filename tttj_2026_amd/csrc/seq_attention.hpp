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

template <typename T, int HD, int RW, int KW, int KT, bool PAGED>
__global__ __launch_bounds__(64 * RW * KW, HD <= 128 && RW * KW == 4 ? 2 : 1) void seq_attention_kernel(SeqAttnArgs a) {
  using v2 = typename Num<T>::v2;
  using v8 = typename Num<T>::v8;
  constexpr int R = 32 * RW;
  constexpr int KB = KT / 32;               // 32-key blocks of a tile
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
  const int wr0 = r0 + rw * 32;
  const bool wave_active = wr0 < rows;
  const int block_lo = seq_limit(a, r0 / G, sq.count, keys);  // the first row's
  const int lim_lo = seq_limit(a, min(wr0, rows - 1) / G, sq.count, keys);
  const int lim_hi = min(seq_limit(a, min(wr0 + 31, rows - 1) / G, sq.count, keys), kend);
  const int r = min(wr0 + col, rows - 1);
  const int tok = r / G, head = hkv * G + r - tok * G;
  const int lim = seq_limit(a, tok, sq.count, keys);

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

  // Paged: lane l holds the page of 16-key group l % (KT / 16) of a tile.
  auto tile_pages = [&](int t0) -> int {
    const int key = min(t0 + 16 * (lane & (KT / 16 - 1)), max(keys - 1, 0));
    return a.table[sq.seq * a.table_row + (key >> a.page_shift)];
  };
  // 16-key groups of a tile whose page number lies outside the cache; their keys are not read and count as NaN.
  auto bad_groups = [&](int pe, int t0) -> uint32_t {
    return (uint32_t)__ballot((uint32_t)pe >= (uint32_t)a.pages && t0 + 16 * lane < keys) & ((1u << (KT / 16)) - 1);
  };
  auto issue_tile = [&](int t0, int st, int pe) {
#pragma unroll
    for (int p = 0; p < PG; ++p) {
      const int g0 = rw * WROWS + p * 16;
      const int t = t0 + g0;
      const int n = min(max(keys - t, 0), 16);
      const T *kp, *vp;
      if constexpr (PAGED) {
        const int e = __builtin_amdgcn_readlane(pe, g0 / 16);
        const int page = (uint32_t)e < (uint32_t)a.pages ? e : 0;
        const int in = t & ((1 << a.page_shift) - 1);
        kp = kh + page * a.k_page + in * a.k_row;
        vp = vh + page * a.v_page + in * a.v_row;
      } else {
        kp = kh + (int64_t)(sq.first + min(t, keys - 1)) * a.k_row;
        vp = vh + (int64_t)(sq.first + min(t, keys - 1)) * a.v_row;
      }
      const __amdgpu_buffer_rsrc_t kr = buffer_rsrc(kp, n == 0 ? 0 : (uint32_t)((n - 1) * (int)a.k_row + hd) * 2);
      const __amdgpu_buffer_rsrc_t vr = buffer_rsrc(vp, n == 0 ? 0 : (uint32_t)((n - 1) * (int)a.v_row + hd) * 2);
#pragma unroll
      for (int c = 0; c < CPG; ++c)
        lds_copy16_buf(kr, koff[c], reinterpret_cast<half*>(sk + st * TILE + (g0 + c * RPC) * HD));
#pragma unroll
      for (int c = 0; c < CPG; ++c)
        lds_copy16_buf(vr, voff[c], reinterpret_cast<half*>(sv + st * TILE + (g0 + c * RPC) * HD));
    }
  };
  // This wave's copies have landed; V rows of keys behind the last are cleared (0 times whatever lay there would
  // not be 0), and the waves of the block meet.
  auto land_tile = [&](int t0, int st) {
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("" ::: "memory");
    const int g0 = rw * WROWS;
    const int n = max(keys - (t0 + g0), 0);
    if (n < WROWS) {
      for (int e = n * CH + lane; e < WROWS * CH; e += 64)
        *reinterpret_cast<u32x4*>(sv + st * TILE + g0 * HD + e * 8) = u32x4{0u, 0u, 0u, 0u};
      __builtin_amdgcn_s_waitcnt(0xC07F);
      asm volatile("" ::: "memory");
    }
    if constexpr (RW > 1) raw_barrier();
  };

  if (hd < HD) {
    for (int e = tid; e < 4 * KW * TILE / 8; e += 64 * RW * KW)
      reinterpret_cast<u32x4*>(seq_lds)[e] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
  }

  v8 qf[KSTEPS];
  {
    const T* qp = static_cast<const T*>(a.q) + (int64_t)(sq.first + tok) * a.q_row + head * a.q_head;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      if (16 * kk + 8 * hf < hd) qf[kk] = *reinterpret_cast<const v8*>(qp + 16 * kk + 8 * hf);
      else qf[kk] = __builtin_bit_cast(v8, u32x4{0u, 0u, 0u, 0u});
    }
  }

  const float c2 = a.scale_log2, lazy = kSeqLazy / a.scale_log2;
  const int vrow = 4 * hf + ((lane >> 2) & 3);       // row, chunk and half chunk of a transposing read
  const int vchunk = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
  floatx16 o[DB];
  float m_ref, l_run, mc, thr;

  // A key that some rows of a tile see and others do not may hold infinities or NaN in V, and 0 times those would
  // reach the rows that do not see it.  If a wave's result is not finite, the block repeats its pass with `careful`
  // set: such values are then added to the rows that see them and taken out of the tile.
  bool careful = false;
  for (;;) {
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    m_ref = -INFINITY;  // the maximum that the sums are relative to, in units of the raw scores
    l_run = 0.f;        // this lane's half of the row's sum
    mc = 0.f;           // m_ref c log2(e) - 7
    thr = -INFINITY;    // a tile maximum above this moves m_ref

    int pe = 0, pe_next = 0;
    if (grp < ntiles) {
      const int t0 = kbeg + grp * KT;
      if constexpr (PAGED) {
        pe = tile_pages(t0);
        pe_next = tile_pages(t0 + KW * KT);
      }
      issue_tile(t0, 0, pe);
    }
    land_tile(kbeg + grp * KT, 0);
    const int rounds = RW == 1 ? (ntiles - grp + KW - 1) / KW : (ntiles + KW - 1) / KW;
    for (int round = 0; round < rounds; ++round) {
      const int t = round * KW + grp;
      const int t0 = kbeg + t * KT;
      const int st = round & 1;
      const uint32_t bad = PAGED ? bad_groups(pe, t0) : 0;
      if (t + KW < ntiles) {
        const int pn = pe_next;
        if constexpr (PAGED) pe_next = tile_pages(t0 + 2 * KW * KT);
        issue_tile(t0 + KW * KT, st ^ 1, pn);
        pe = pn;
      }
      if (careful) {
        if (t < ntiles && wave_active && t0 + KT > block_lo && t0 < lim_hi) {
#pragma unroll 1
          for (int key = 0; key < KT; ++key)
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const int d = 32 * i + 8 * (e >> 2) + 4 * hf + (e & 3);
                const T x = sv[st * TILE + key * HD + vseg<HD>(key, d >> 3) * 8 + (d & 7)];
                const uint16_t bits = __builtin_bit_cast(uint16_t, x);
                if ((bits & Num<T>::kExp) == Num<T>::kExp && t0 + key < lim) o[i][e] += (float)x;
              }
        }
        if constexpr (RW > 1) __syncthreads();
        if (t < ntiles && t0 + KT > block_lo) {
          for (int e = lane; e < WROWS * HD; e += 64) {
            T* const p = sv + st * TILE + rw * WROWS * HD + e;
            if ((__builtin_bit_cast(uint16_t, *p) & Num<T>::kExp) == Num<T>::kExp) *p = (T)0.f;
          }
        }
        if constexpr (RW > 1) __syncthreads();
      }
      if (wave_active && t0 < lim_hi) {
        floatx16 s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const int row = kb * 32 + col;
#pragma unroll
          for (int e = 0; e < 16; ++e) s[kb][e] = 0.f;
#pragma unroll
          for (int kk = 0; kk < KSTEPS; ++kk) {
            const v8 x = *reinterpret_cast<const v8*>(sk + st * TILE + row * HD + kswz<HD>(row, 2 * kk + hf) * 8);
            s[kb] = Num<T>::mfma(x, qf[kk], s[kb]);
          }
        }
        if (t0 + KT > lim_lo || bad != 0) {
          const int rem = lim - t0 - 4 * hf;
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              if ((bad >> (2 * kb + (j >> 3))) & 1u) s[kb][j] = __builtin_nanf("");
              s[kb][j] = 32 * kb + 8 * (j >> 2) + (j & 3) < rem ? s[kb][j] : -INFINITY;
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[kb][j]);
        const float mt = xhalf_max(mx);
        if (__builtin_amdgcn_ballot_w64(mt > thr) != 0) {
          const float m_new = fmaxf(m_ref, mt);
          const bool none = m_new == -INFINITY;  // no key of this row so far: o and l are 0
          const float corr = none ? 1.f : __builtin_amdgcn_exp2f((m_ref - m_new) * c2);
          m_ref = m_new;
          mc = none ? 0.f : m_new * c2 - kSeqShift;
          thr = none ? -INFINITY : m_new + lazy;
          l_run *= corr;
#pragma unroll
          for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] *= corr;
        }
        v8 p16[KB][2];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[kb][j], c2, -mc));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s[kb][j + 1], c2, -mc));
            const v2 pp = {(T)p0, (T)p1};
            l_run = Num<T>::add2(pp, l_run);
            p16[kb][j >> 3][j & 7] = pp[0];
            p16[kb][j >> 3][(j & 7) + 1] = pp[1];
          }
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              // keys 32 kb + 16 c + 4 hf + {0..3} and 8 further: the order of the lane's probabilities
              const int ra = 32 * kb + 16 * c + vrow;
              using lds4 = __attribute__((address_space(3))) shortx4;
              const T* pa = sv + st * TILE + ra * HD + vseg<HD>(ra, 4 * i + vchunk) * 8 + 4 * (lane & 1);
              const shortx4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(pa));
              const shortx4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(pa + 8 * HD));
              const shortx8 x = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
              o[i] = Num<T>::mfma(__builtin_bit_cast(v8, x), p16[kb][c], o[i]);
            }
      }
      if (round + 1 < rounds) land_tile(t0 + KW * KT, st ^ 1);
    }
    if (careful || !a.causal || sq.count == 1) break;
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) z = fmaf(o[i][e], 0.f, z);
    const bool odd = __builtin_amdgcn_ballot_w64(z != 0.f) != 0;  // 0 times infinity or NaN is NaN
    if constexpr (RW > 1) careful = __syncthreads_or(odd);
    else careful = odd;
    if (!careful) break;
  }

  if constexpr (KW > 1) {
    // [group - 1][wave of the group][value][lane]: O, the maximum in log2 units and this lane's half of the sum
    constexpr int NV = DB * 16 + 2;
    float* const mrg = reinterpret_cast<float*>(seq_lds);
    __syncthreads();
    if (grp > 0) {
      float* p = mrg + (size_t)((grp - 1) * RW + rw) * NV * 64 + lane;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) p[(i * 16 + e) * 64] = o[i][e];
      p[(NV - 2) * 64] = m_ref;
      p[(NV - 1) * 64] = l_run;
    }
    __syncthreads();
    if (grp > 0) return;
#pragma unroll 1
    for (int g = 0; g < KW - 1; ++g) {
      const float* p = mrg + (size_t)(g * RW + rw) * NV * 64 + lane;
      const float m_g = p[(NV - 2) * 64], l_g = p[(NV - 1) * 64];
      const float m_new = fmaxf(m_ref, m_g);
      // a part without a maximum saw no key (its sum, 0, is then its weight) or only NaN (NaN is)
      const float c0 = m_ref == -INFINITY ? l_run : __builtin_amdgcn_exp2f((m_ref - m_new) * c2);
      const float c1 = m_g == -INFINITY ? l_g : __builtin_amdgcn_exp2f((m_g - m_new) * c2);
      l_run = l_run * c0 + l_g * c1;
      m_ref = m_new;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = o[i][e] * c0 + p[(i * 16 + e) * 64] * c1;
    }
  }

  if (wr0 + col >= rows) return;
  const float l = xhalf_sum(l_run);
  const int64_t orow = (int64_t)(sq.first + tok) * a.heads + head;
  if (lim > a.chunk) {  // this row's keys lie in several parts
    float* dst = a.part_o + ((int64_t)split * a.tokens * a.heads + orow) * hd;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (32 * i + 8 * g < hd)
          *reinterpret_cast<floatx4*>(dst + 32 * i + 8 * g + 4 * hf) =
              floatx4{o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]};
    if (hf == 0) a.part_ml[(int64_t)split * a.tokens * a.heads + orow] = make_float2(m_ref * c2, l);
    return;
  }
  if (split > 0) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;  // no key: zeros
  T* dst = static_cast<T*>(a.out) + orow * hd;
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (32 * i + 8 * g < hd) {
        typedef T v4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<v4*>(dst + 32 * i + 8 * g + 4 * hf) =
            v4{(T)(o[i][4 * g] * inv), (T)(o[i][4 * g + 1] * inv), (T)(o[i][4 * g + 2] * inv),
               (T)(o[i][4 * g + 3] * inv)};
      }
}

}  // namespace tt
