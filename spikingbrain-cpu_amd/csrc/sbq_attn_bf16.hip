// sbq_attn_bf16.hip - attention over a cache of bf16 (sbq_attn.h): 2-byte products where
// the queries are of the same type, fp32 products for fp32 queries and for
// rows that 16-byte loads cannot read.
#include "sbq_attn.h"

namespace sbq {

int launch_attn_bf16(const AttnArgs& a, bool m16, int DP, int mode, int RT, float* weight, hipStream_t st) {
  return m16 ? launch_attn_ct<XT_BF16, true>(a, DP, mode, RT, weight, st)
             : launch_attn_ct<XT_BF16, false>(a, DP, mode, RT, weight, st);
}

}  // namespace sbq
