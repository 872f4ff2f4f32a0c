// The write of new keys and values into a paged cache in 8 bits, with a power of two as scale for each block of tokens
// and head.
//
// A block holds x as e4m3(x 2^-e) and e, the smallest with max |x| <= 448 2^e.  A power of two: e4m3 has an exponent of
// its own, so a finer scale would gain no bit; a scale that grows with a later token moves what is stored by its exponent
// (exact but for values that become subnormal); and the attention widens the product to 16 bits in one instruction.
#include "cache_checks.hpp"
#include "seq_attention.hpp"

namespace tt {

struct Append8Args {
  const uint16_t *k, *v;
  uint8_t *k_cache, *v_cache, *k_scales, *v_scales;
  const int32_t *starts, *lengths, *table;
  int64_t k_row, k_head, v_row, v_head, kc_page, kc_row, kc_head, vc_page, vc_row, vc_head;
  int64_t s_page, s_block, s_head, table_row;
  int tokens, batch, heads, chunks;  // a row: `chunks` times 8 values
  uint32_t by_chunks;                // 2^32 / chunks, rounded up
  int pages, table_pages, page_shift, block_shift, units;
};

template <typename T>
struct Raw16;
template <>
struct Raw16<half> {
  static constexpr float kTop = 0x1.ep15f;  // 15/16 of the way to the next power of two: rounded up it would be none of T's
  static __device__ __forceinline__ float get(uint32_t x, int i) {
    return (float)__builtin_bit_cast(half, (uint16_t)(x >> (16 * i)));
  }
};
template <>
struct Raw16<bf16> {
  static constexpr float kTop = 0x1.ep127f;
  static __device__ __forceinline__ float get(uint32_t x, int i) {
    return __builtin_bit_cast(float, i == 0 ? x << 16 : x & 0xffff0000u);
  }
};

// The magnitudes of two values, 0 where one is infinite or NaN.
template <typename T>
__device__ __forceinline__ uint32_t finite_pair(uint32_t x) {
  constexpr uint32_t kCarry = (0x8000u - Num<T>::kExp) * 0x10001u;  // an exponent of ones carries into the sign
  x &= 0x7fff7fffu;
  return x & ~((((x + kCarry) >> 15) & 0x10001u) * 0xffffu);
}

__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// Eight values times `factor` in e4m3.
template <typename T>
__device__ __forceinline__ u32x2 narrow8(u32x4 x, float factor) {
  const float top = Raw16<T>::kTop * factor;
  u32x2 y;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = x[2 * i + j / 2], bits = (w >> (16 * (j & 1))) & 0x7fff;
      f[j] = __builtin_amdgcn_fmed3f(Raw16<T>::get(w, j & 1) * factor, -top, top);
      if (bits >= Num<T>::kExp) f[j] = __builtin_nanf("");
    }
    int z = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    y[i] = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], z, true);
  }
  return y;
}

// Eight values of e4m3 times `factor`, in e4m3.
__device__ __forceinline__ u32x2 rescale8(u32x2 x, float factor) {
  u32x2 y;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int z = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_cvt_f32_fp8(x[i], 0) * factor,
                                                  __builtin_amdgcn_cvt_f32_fp8(x[i], 1) * factor, 0, false);
    y[i] = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_cvt_f32_fp8(x[i], 2) * factor,
                                           __builtin_amdgcn_cvt_f32_fp8(x[i], 3) * factor, z, true);
  }
  return y;
}

// W waves per (block of tokens, half, head).  Sequence b's blocks begin at unit floor(starts[b] / block) + 2 b, which
// leaves it at least as many as its n new tokens touch (n / block + 2), so no table of them is needed.  Up to 8 pieces of
// 16 bytes a lane stay in registers between the maximum and the rounding; what is beyond is read again.  Bound by HBM:
// 36207 tokens on 8 heads of 128 47.6 us, 4.7 TB/s read and written.  (The launch bound is what makes the compiler widen
// pieces one by one: it took 228 registers for 55 without it, and 97 us.)
template <typename T, int W>
__global__ __launch_bounds__(256, 4) void cache_append8_kernel(Append8Args a) {
  __shared__ uint32_t s_max[4];
  constexpr int KEPT = 8;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int at = W > 1 ? (int)threadIdx.x : (int)threadIdx.x & 63;  // of the 64 W lanes
  const int task = W > 1 ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave;
  const int head = task % a.heads, rest = task / a.heads;
  const bool is_v = rest & 1;
  const int unit = rest >> 1;
  if (unit >= a.units) return;
  int seq = unit, first = unit, count = 1, number = 0;
  const int shift = a.block_shift;
  if (a.starts != nullptr) {
    const auto unit_of = [&](int b) { return (seq_start(a.starts, b, a.tokens) >> shift) + 2 * b; };
    seq = seq_search(a.batch, unit, unit_of);
    number = unit - unit_of(seq);
    first = seq_start(a.starts, seq, a.tokens);
    count = seq_start(a.starts, seq + 1, a.tokens) - first;
  }
  // This block's positions lo ... hi - 1 are new; those before begin are older tokens.
  const int64_t length = a.lengths[seq], begin = length - count, from = begin > 0 ? begin : 0;
  const int64_t base = ((from >> shift) + number) << shift;
  const int64_t held = (int64_t)a.table_pages << a.page_shift;
  const int64_t lo = base > from ? base : from, end = length < held ? length : held;
  const int64_t hi = base + (1 << shift) < end ? base + (1 << shift) : end;
  if (number < 0 || lo >= hi) return;
  const int page = a.table[seq * a.table_row + (base >> a.page_shift)];
  if ((uint32_t)page >= (uint32_t)a.pages) return;
  const int in = (int)base & ((1 << a.page_shift) - 1);

  const int64_t row = is_v ? a.v_row : a.k_row, to_row = is_v ? a.vc_row : a.kc_row;
  const uint16_t* const x = (is_v ? a.v + head * a.v_head : a.k + head * a.k_head) + (first + (lo - begin)) * row;
  uint8_t* const block = is_v ? a.v_cache + page * a.vc_page + in * a.vc_row + head * a.vc_head
                              : a.k_cache + page * a.kc_page + in * a.kc_row + head * a.kc_head;
  uint8_t* const scale = (is_v ? a.v_scales : a.k_scales) + page * a.s_page + (in >> shift) * a.s_block + head * a.s_head;
  const int older = (int)(lo - base), pieces = (int)(hi - lo) * a.chunks;
  const uint32_t old = older > 0 ? *scale : 0;
  const auto place = [&](int piece) -> int2 {  // its token of the block's new ones, and its first value
    const int t = __umulhi((uint32_t)piece, a.by_chunks);
    return make_int2(t, (piece - t * a.chunks) * 8);
  };
  const auto load = [&](int piece) -> u32x4 {
    const int2 p = place(piece);
    return *reinterpret_cast<const u32x4*>(x + p.x * row + p.y);
  };
  u32x4 kept[KEPT];
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < KEPT; ++i) {
    kept[i] = u32x4{0u, 0u, 0u, 0u};
    if (at + 64 * W * i < pieces) kept[i] = load(at + 64 * W * i);
  }
#pragma unroll
  for (int i = 0; i < KEPT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) most = max_pair(most, finite_pair<T>(kept[i][j]));
  for (int piece = at + 64 * W * KEPT; piece < pieces; piece += 64 * W) {
    const u32x4 y = load(piece);
#pragma unroll
    for (int j = 0; j < 4; ++j) most = max_pair(most, finite_pair<T>(y[j]));
  }
  most = wave_max_int(max(most & 0xffffu, most >> 16));
  if constexpr (W > 1) {
    s_max[wave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) most = max(most, s_max[w]);
  }
  // 1.75 2^8 = 448 is the largest of e4m3.
  const uint32_t bits = __builtin_bit_cast(uint32_t, Raw16<T>::get(most, 0));
  const int need = max((int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), 0);
  const int e = max(need, (int)old);
  const float factor = __builtin_bit_cast(float, e >= 254 ? 0x400000u : (uint32_t)(254 - e) << 23);  // 2^(127 - e)
  const auto store = [&](int piece, u32x4 y) {
    const int2 p = place(piece);
    *reinterpret_cast<u32x2*>(block + (older + p.x) * to_row + p.y) = narrow8<T>(y, factor);
  };
#pragma unroll
  for (int i = 0; i < KEPT; ++i)
    if (at + 64 * W * i < pieces) store(at + 64 * W * i, kept[i]);
  for (int piece = at + 64 * W * KEPT; piece < pieces; piece += 64 * W) store(piece, load(piece));
  if (older > 0 && e > (int)old) {
    const float less = __builtin_bit_cast(float, (uint32_t)(127 - min(e - (int)old, 126)) << 23);
    for (int piece = at; piece < older * a.chunks; piece += 64 * W) {
      const int2 p = place(piece);
      u32x2* const y = reinterpret_cast<u32x2*>(block + p.x * to_row + p.y);
      *y = rescale8(*y, less);
    }
  }
  if (at == 0 && (older == 0 || e > (int)old)) *scale = (uint8_t)e;
}

template <typename T>
static int launch_append8(const Append8Args& a, bool large, hipStream_t stream) {
  const int64_t tasks = (int64_t)a.units * 2 * a.heads, blocks = large ? tasks : (tasks + 3) / 4;
  TT_REQUIRE(tasks < (1LL << 31) && blocks * 256 < (1LL << 32), "cache_append: %lld blocks of tokens are more than one launch takes",
             (long long)tasks);
  if (large) hipLaunchKernelGGL((cache_append8_kernel<T, 4>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((cache_append8_kernel<T, 1>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return launch_status("cache_append8_kernel");
}

}  // namespace tt

extern "C" int tt_cache_append8(const tt_cache_rows8* args, void* stream) {
  using namespace tt;
  TT_ARGS(tt_cache_rows8, "cache_append");
  TT_CHECK(check_heads("cache_append", c.tokens, c.batch, c.kv_heads, c.kv_heads, c.head_dim, c.dtype));
  TT_CHECK(check_head8("cache_append", c.head_dim));
  TT_CHECK(check_pages("cache_append", c.pages, c.page_size, c.table_pages));
  TT_CHECK(check_block("cache_append", c.block, c.page_size));
  if (c.tokens == 0 || c.batch == 0) return TT_OK;
  TT_REQUIRE(c.k && c.v && c.k_cache && c.v_cache && c.table && c.lengths, "cache_append: null pointer");
  TT_REQUIRE(c.starts != nullptr || c.tokens == c.batch, "cache_append: %d tokens for %d sequences without starts",
             c.tokens, c.batch);
  TT_CHECK(check_rows("cache_append: k", c.k, c.k_row, c.k_head));
  TT_CHECK(check_rows("cache_append: v", c.v, c.v_row, c.v_head));
  TT_CHECK(check_rows8("cache_append: k_cache", c.k_cache, c.kc_page, c.kc_row, c.kc_head));
  TT_CHECK(check_rows8("cache_append: v_cache", c.v_cache, c.vc_page, c.vc_row, c.vc_head));
  TT_CHECK(check_scales("cache_append", c));
  TT_CHECK(check_apart("cache_append: k_cache", "pages", c.kc_page, c.pages));
  TT_CHECK(check_apart("cache_append: v_cache", "pages", c.vc_page, c.pages));
  TT_CHECK(check_apart("cache_append: k_cache", "rows", c.kc_row, c.page_size));
  TT_CHECK(check_apart("cache_append: v_cache", "rows", c.vc_row, c.page_size));
  TT_CHECK(check_apart("cache_append: k_cache", "heads", c.kc_head, c.kv_heads));
  TT_CHECK(check_apart("cache_append: v_cache", "heads", c.vc_head, c.kv_heads));
  TT_CHECK(check_apart("cache_append: scales", "pages", c.s_page, c.pages));
  TT_CHECK(check_apart("cache_append: scales", "blocks", c.s_block, c.page_size / c.block));
  TT_CHECK(check_apart("cache_append: scales", "heads", c.s_head, c.kv_heads));
  TT_REQUIRE(c.table_row >= 0, "cache_append: table_row %lld", (long long)c.table_row);
  Append8Args a{};
  a.k = static_cast<const uint16_t*>(c.k), a.v = static_cast<const uint16_t*>(c.v);
  a.k_cache = static_cast<uint8_t*>(c.k_cache), a.v_cache = static_cast<uint8_t*>(c.v_cache);
  a.k_scales = c.k_scales, a.v_scales = c.v_scales;
  a.starts = c.starts, a.lengths = c.lengths, a.table = c.table;
  a.k_row = c.k_row, a.k_head = c.k_head, a.v_row = c.v_row, a.v_head = c.v_head;
  a.kc_page = c.kc_page, a.kc_row = c.kc_row, a.kc_head = c.kc_head;
  a.vc_page = c.vc_page, a.vc_row = c.vc_row, a.vc_head = c.vc_head;
  a.s_page = c.s_page, a.s_block = c.s_block, a.s_head = c.s_head, a.table_row = c.table_row;
  a.tokens = c.tokens, a.batch = c.batch, a.heads = c.kv_heads, a.chunks = c.head_dim / 8;
  a.by_chunks = (uint32_t)(((1ull << 32) + a.chunks - 1) / a.chunks);
  a.pages = c.pages, a.table_pages = c.table_pages, a.page_shift = __builtin_ctz(c.page_size);
  a.block_shift = __builtin_ctz(c.block);
  const int64_t units = c.starts == nullptr ? c.batch : (int64_t)(c.tokens >> a.block_shift) + 2 * (int64_t)c.batch;
  TT_REQUIRE(units < (1LL << 30), "cache_append: %lld blocks of tokens are more than one launch takes", (long long)units);
  a.units = (int)units;
  const bool large = (int64_t)c.block * a.chunks > 512;  // pieces of a block: more than one wave keeps
  return c.dtype == TT_FP16 ? launch_append8<half>(a, large, (hipStream_t)stream)
                            : launch_append8<bf16>(a, large, (hipStream_t)stream);
}
