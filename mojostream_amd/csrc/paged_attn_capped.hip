// Paged attention with capped scores, over fp32, bf16 and fp16 pools.
#include "paged_attn.h"

namespace ms {

int launch_attn_capped(PagedAttnArgs &a, ms_paged_batch *b, int dtype, int hd, int most, hipStream_t st) {
  if (dtype == MS_KV_F32) return launch_dims<MS_KV_F32, true>(a, b, hd, most, st);
  if (dtype == MS_KV_BF16) return launch_dims<MS_KV_BF16, true>(a, b, hd, most, st);
  return launch_dims<MS_KV_F16, true>(a, b, hd, most, st);
}

}  // namespace ms
