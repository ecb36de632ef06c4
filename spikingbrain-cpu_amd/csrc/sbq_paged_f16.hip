// sbq_paged_f16.hip - the attention over an fp16 cache in pages (sbq_paged.h).
#include "sbq_paged.h"

namespace sbq {

int launch_paged_attn_f16(const PagedArgs& a, int DP, dim3 grid, hipStream_t st) {
  return a.qt == XT_F32 ? launch_paged_types<XT_F16, XT_F32>(a, DP, grid, st) : launch_paged_types<XT_F16, XT_F16>(a, DP, grid, st);
}

}  // namespace sbq
