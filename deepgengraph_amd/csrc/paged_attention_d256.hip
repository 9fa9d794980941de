// Attention over a paged cache at head_dim 256 (kernels and launch rules in paged_attention.h).
#include "paged_attention.h"

namespace dgg_paged {

void launch_d256(const PagedParams& p, bool bf16, hipStream_t st) {
  if (bf16) launch_paged<BF16, 256>(p, st);
  else launch_paged<F16, 256>(p, st);
}

}  // namespace dgg_paged
