// The attention over a paged cache for rows of bfloat16.
#include "paged_attend.cuh"

namespace certex_b200 {

void launch_attend_bf16(const AttendParams& p, int64_t blocks, cudaStream_t s)
{
  launch_half<__nv_bfloat16>(p, blocks, s);
  if (!p.cluster) { launch_join<__nv_bfloat16>(p, s); }
}

}  // namespace certex_b200
