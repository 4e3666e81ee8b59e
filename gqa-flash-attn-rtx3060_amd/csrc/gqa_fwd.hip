// gqa_fwd.hip — the single-pass kernel (gqa_fwd_kernel.hpp) as
// gqa_flash_attn and paged_attention launch it without changed scores.
#include "gqa_fwd_kernel.hpp"

namespace gqa {

hipError_t launch_fwd(const FwdParams& p, int dtype, hipStream_t stream, const ScoreMod* mod) {
  if (mod != nullptr) return launch_fwd_mod(p, dtype, stream, *mod);
  return launch_fwd_pg<0>(p, dtype, stream);
}

hipError_t launch_paged_fwd(const FwdParams& p, int dtype, hipStream_t stream, const ScoreMod* mod) {
  if (mod != nullptr) return launch_fwd_mod(p, dtype, stream, *mod);
  return launch_paged_fwd_p(p, dtype, stream);
}

}  // namespace gqa
