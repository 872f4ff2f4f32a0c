// seq_attention_kernel over a cache in 8 bits, for head_dim above 128.
#include "seq_launch.hpp"

namespace tt {

int launch_seq8_attention_wide(const SeqAttnArgs& a, SeqShape shape, int dtype, hipStream_t stream) {
  return launch_seq8_hd<256>(a, shape, dtype, stream);
}

}  // namespace tt
