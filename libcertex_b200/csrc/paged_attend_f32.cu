// The attention over a paged cache for rows of float32.
#include "paged_attend.cuh"

namespace certex_b200 {

void launch_attend_f32(const AttendParams& p, int64_t blocks, cudaStream_t s)
{
  if (p.dim <= 64) {
    launch_float<64>(p, blocks, s);
  } else if (p.dim <= 96) {
    launch_float<96>(p, blocks, s);
  } else if (p.dim <= 128) {
    launch_float<128>(p, blocks, s);
  } else {
    launch_float<256>(p, blocks, s);
  }
  if (!p.cluster) { launch_join<float>(p, s); }
}

}  // namespace certex_b200
