// The streaming kernel (reach_stream.h) over bf16 pools: an object of its own, to be built beside the others.
#include "reach_stream.h"

namespace pia {

int launch_reach_stream_bf16(const reach::Args& a, int64_t tokens, hipStream_t s) {
  return reach_stream::launch_dtype<PIA_DTYPE_BF16>(a, tokens, s);
}

}  // namespace pia
