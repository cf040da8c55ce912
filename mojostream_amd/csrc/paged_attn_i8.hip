// Paged attention over pools of 8-bit integers.
#include "paged_attn.h"

namespace ms {

int launch_attn_i8(PagedAttnArgs &a, ms_paged_batch *b, int hd, int most, hipStream_t st) {
  return a.cap_to != 0.f ? launch_dims<MS_KV_I8, true>(a, b, hd, most, st)
                        : launch_dims<MS_KV_I8, false>(a, b, hd, most, st);
}

}  // namespace ms
