// Attention over a paged cache at head_dim 64 (kernels and launch rules in paged_attention.h).
#include "paged_attention.h"

namespace dgg_paged {

void launch_d64(const PagedParams& p, bool bf16, hipStream_t st) {
  if (bf16) launch_paged<BF16, 64>(p, st);
  else launch_paged<F16, 64>(p, st);
}

}  // namespace dgg_paged
