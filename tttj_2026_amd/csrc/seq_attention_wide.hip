// seq_attention_kernel for head_dim above 128 (one wave per SIMD; of its 512 registers the compiler keeps 128
// accumulator floats per lane in AGPRs).
#include "seq_launch.hpp"

namespace tt {

int launch_seq_attention_wide(const SeqAttnArgs& a, bool paged, SeqShape shape, int dtype, hipStream_t stream) {
  return launch_seq_hd<256>(a, paged, shape, dtype, stream);
}

}  // namespace tt
