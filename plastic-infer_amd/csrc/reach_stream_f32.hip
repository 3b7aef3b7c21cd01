// The streaming kernel (reach_stream.h) over f32 pools: an object of its own, to be built beside the others.
#include "reach_stream.h"

namespace pia {

int launch_reach_stream_f32(const reach::Args& a, int64_t tokens, hipStream_t s) {
  return reach_stream::launch_dtype<PIA_DTYPE_F32>(a, tokens, s);
}

// the same for all types: whole waves of the card, two pieces of 16 rows each
int64_t reach_stream_pref_bytes() { return reach_stream::PREF_BYTES; }
int64_t reach_stream_parts_bytes(int D) {
  const int DP = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  return reach_stream::resident_waves() * 2 * 16 * (DP + 2) * int64_t(sizeof(float));
}

}  // namespace pia
