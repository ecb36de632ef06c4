// sbq_paged_f32.hip - the attention over an fp32 cache in pages (sbq_paged.h).
#include "sbq_paged.h"

namespace sbq {

int launch_paged_attn_f32(const PagedArgs& a, int DP, unsigned grid, hipStream_t st) {
  return launch_paged_types<XT_F32, 1, 1>(a, DP, grid, st);
}

}  // namespace sbq
