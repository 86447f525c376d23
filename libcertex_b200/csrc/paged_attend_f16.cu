// The attention over a paged cache for rows of float16.
#include "paged_attend.cuh"

namespace certex_b200 {

void launch_attend_f16(const AttendParams& p, int64_t blocks, cudaStream_t s)
{
  launch_half<__half>(p, blocks, s);
  if (!p.cluster) { launch_join<__half>(p, s); }
}

}  // namespace certex_b200
