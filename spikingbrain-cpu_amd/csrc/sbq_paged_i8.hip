// sbq_paged_i8.hip - the attention over an int8 cache in pages (sbq_paged.h).
#include "sbq_paged.h"

namespace sbq {

int launch_paged_attn_i8(const PagedArgs& a, int DP, unsigned grid, hipStream_t st) {
  return a.qt == XT_F32 ? launch_paged_types<CT_I8, 2, 2>(a, DP, grid, st) : launch_paged_types<CT_I8, 1, 1>(a, DP, grid, st);
}

}  // namespace sbq
