// seq_attention_kernel over a cache in 8 bits (heads to 128).
#include "seq_launch.hpp"

namespace tt {

int launch_seq8_attention(const SeqAttnArgs& a, SeqShape shape, int dtype, hipStream_t stream) {
  if (a.head_dim > 128) return launch_seq8_attention_wide(a, shape, dtype, stream);
  if (a.head_dim > 64) return launch_seq8_hd<128>(a, shape, dtype, stream);
  return launch_seq8_hd<64>(a, shape, dtype, stream);
}

}  // namespace tt
