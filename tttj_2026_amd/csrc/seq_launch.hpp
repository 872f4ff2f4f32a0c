// Host side of seq_attention.hpp: the launch of one instantiation, shared by seq_attention.hip (head_dim up to
// 128) and seq_attention_wide.hip (up to 256).
#pragma once

#include "cache_checks.hpp"
#include "seq_attention.hpp"

#include <atomic>

namespace tt {

// Blocks of 128 rows on four waves; of 32 rows, for single tokens and few drafted ones, whose keys are shared by one
// or two waves; and of 32 rows with as many waves as the LDS holds tiles for, where blocks are few.
enum class SeqShape { kWide, kNarrow, kDeep };

// Waves of a block of 32 rows on heads up to `hd`.
constexpr int seq_waves(SeqShape shape, int hd) {
  return shape == SeqShape::kDeep ? (hd <= 64 ? 8 : hd <= 128 ? 4 : 2) : (hd <= 128 ? 2 : 1);
}

template <typename T, int HD, int RW, int KW, int KT, bool PAGED, bool C8 = false, int NH = 1>
int launch_seq(const SeqAttnArgs& a, hipStream_t stream) {
  // K and V, two tiles deep (narrow blocks over an 8-bit cache hold its bytes); the groups are joined there.
  constexpr int tiles =
      2 * 2 * KW * KT * HD * NH * (C8 && RW == 1 ? 1 : (int)sizeof(T)) + (C8 && RW > 1 ? 2 * 16 * RW * HD : 0);
  constexpr int joined = KW == 1 ? 0 : KW * (HD / 8 * 64 * 16 + 32 * 8 + 4);
  constexpr int lds = tiles > joined ? tiles : joined;
  static std::atomic<uint64_t> ready{0};  // devices whose limit of dynamic LDS is raised
  int dev = 0;
  TT_HIP(hipGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if ((ready.load(std::memory_order_relaxed) & bit) == 0) {
    TT_HIP(hipFuncSetAttribute((const void*)seq_attention_kernel<T, HD, RW, KW, KT, PAGED, C8, NH>,
                               hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const int64_t blocks = (int64_t)a.slots * (a.kv_heads / NH);
  constexpr int threads = 64 * RW * KW * NH;
  TT_REQUIRE(blocks * threads < (1LL << 32), "attention: %lld blocks are more than one launch takes",
             (long long)blocks);
  hipLaunchKernelGGL((seq_attention_kernel<T, HD, RW, KW, KT, PAGED, C8, NH>), dim3((unsigned)blocks), dim3(threads), lds,
                     stream, a);
  return launch_status("seq_attention_kernel");
}

template <int HD, typename T>
int launch_seq_type(const SeqAttnArgs& a, bool paged, SeqShape shape, hipStream_t stream) {
  if (!paged) return launch_seq<T, HD, 4, 1, 64, false>(a, stream);
  if (shape == SeqShape::kDeep) return launch_seq<T, HD, 1, seq_waves(SeqShape::kDeep, HD), 32, true>(a, stream);
  if (shape == SeqShape::kNarrow) return launch_seq<T, HD, 1, seq_waves(SeqShape::kNarrow, HD), 32, true>(a, stream);
  return launch_seq<T, HD, 4, 1, 64, true>(a, stream);
}

// Over an 8-bit cache: keys of a wave's tile, and waves of a block of 32 rows.
constexpr int seq8_keys(int hd) { return hd <= 128 ? 64 : 32; }
constexpr int seq8_waves(SeqShape shape, int hd) {
  return shape == SeqShape::kDeep ? (hd <= 64 ? 8 : 4) : (hd <= 128 ? 2 : 1);
}

// Heads that lie side by side in a row of the cache and share a narrow block: 256 bytes of them.
inline int seq8_heads(int head_dim, int kv_heads, int64_t k_head, int64_t v_head) {
  if (k_head != head_dim || v_head != head_dim || head_dim > 128 || kv_heads % 2 != 0) return 1;
  return head_dim <= 64 && kv_heads % 4 == 0 ? 4 : 2;
}

template <int HD, typename T>
int launch_seq8_type(const SeqAttnArgs& a, SeqShape shape, hipStream_t stream) {
  if constexpr (HD <= 128) {
    if (shape == SeqShape::kNarrow) {
      const int heads = seq8_heads(a.head_dim, a.kv_heads, a.k_head, a.v_head);
      if constexpr (HD <= 64)
        if (heads == 4) return launch_seq<T, HD, 1, 1, 64, true, true, 4>(a, stream);
      if (heads == 2) return launch_seq<T, HD, 1, 1, 64, true, true, 2>(a, stream);
    }
  }
  if (shape == SeqShape::kDeep)
    return launch_seq<T, HD, 1, seq8_waves(SeqShape::kDeep, HD), seq8_keys(HD), true, true>(a, stream);
  if (shape == SeqShape::kNarrow)
    return launch_seq<T, HD, 1, seq8_waves(SeqShape::kNarrow, HD), seq8_keys(HD), true, true>(a, stream);
  return launch_seq<T, HD, 4, 1, 64, true, true>(a, stream);
}

template <int HD>
int launch_seq8_hd(const SeqAttnArgs& a, SeqShape shape, int dtype, hipStream_t stream) {
  return dtype == TT_FP16 ? launch_seq8_type<HD, half>(a, shape, stream) : launch_seq8_type<HD, bf16>(a, shape, stream);
}

template <int HD>
int launch_seq_hd(const SeqAttnArgs& a, bool paged, SeqShape shape, int dtype, hipStream_t stream) {
  return dtype == TT_FP16 ? launch_seq_type<HD, half>(a, paged, shape, stream)
                          : launch_seq_type<HD, bf16>(a, paged, shape, stream);
}

int launch_seq_attention_wide(const SeqAttnArgs& a, bool paged, SeqShape shape, int dtype, hipStream_t stream);
int launch_seq8_attention(const SeqAttnArgs& a, SeqShape shape, int dtype, hipStream_t stream);       // 8-bit cache
int launch_seq8_attention_wide(const SeqAttnArgs& a, SeqShape shape, int dtype, hipStream_t stream);  // heads above 128

}  // namespace tt
