// sbq_paged_i8.hip - the attention over an int8 cache in pages (sbq_paged.h).
#include "sbq_paged.h"

namespace sbq {

int launch_paged_attn_i8(const PagedArgs& a, int DP, dim3 grid, hipStream_t st) {
  return a.qt == XT_F32   ? launch_paged_types<CT_I8, XT_F32>(a, DP, grid, st)
         : a.qt == XT_F16 ? launch_paged_types<CT_I8, XT_F16>(a, DP, grid, st)
                          : launch_paged_types<CT_I8, XT_BF16>(a, DP, grid, st);
}

}  // namespace sbq
