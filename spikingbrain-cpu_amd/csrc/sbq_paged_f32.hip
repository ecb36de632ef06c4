// sbq_paged_f32.hip - the attention over an fp32 cache in pages (sbq_paged.h).
#include "sbq_paged.h"

namespace sbq {

int launch_paged_attn_f32(const PagedArgs& a, int DP, dim3 grid, hipStream_t st) {
  return launch_paged_types<XT_F32, XT_F32>(a, DP, grid, st);
}

}  // namespace sbq
