// Host side of seq_attention.hpp: the launch of one instantiation, shared by seq_attention.hip (head_dim up to
// 128) and seq_attention_wide.hip (up to 256).
#pragma once

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

template <typename T, int HD, int RW, int KW, int KT, bool PAGED>
int launch_seq(const SeqAttnArgs& a, hipStream_t stream) {
  constexpr int lds = 2 * 2 * KW * KT * HD * (int)sizeof(T);  // K and V, two tiles deep
  static_assert(KW == 1 || lds >= KW * (HD / 8 * 64 * 16 + 32 * 8 + 4), "the groups are joined in the tiles' LDS");
  static std::atomic<uint64_t> ready{0};  // devices whose limit of dynamic LDS is raised
  int dev = 0;
  TT_HIP(hipGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if ((ready.load(std::memory_order_relaxed) & bit) == 0) {
    TT_HIP(hipFuncSetAttribute((const void*)seq_attention_kernel<T, HD, RW, KW, KT, PAGED>,
                               hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const int64_t blocks = (int64_t)a.slots * a.kv_heads;
  constexpr int threads = 64 * RW * KW;
  TT_REQUIRE(blocks * threads < (1LL << 32), "attention: %lld blocks are more than one launch takes",
             (long long)blocks);
  hipLaunchKernelGGL((seq_attention_kernel<T, HD, RW, KW, KT, PAGED>), dim3((unsigned)blocks), dim3(threads), lds,
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

template <int HD>
int launch_seq_hd(const SeqAttnArgs& a, bool paged, SeqShape shape, int dtype, hipStream_t stream) {
  return dtype == TT_FP16 ? launch_seq_type<HD, half>(a, paged, shape, stream)
                          : launch_seq_type<HD, bf16>(a, paged, shape, stream);
}

int launch_seq_attention_wide(const SeqAttnArgs& a, bool paged, SeqShape shape, int dtype, hipStream_t stream);

}  // namespace tt
