// gqa_fwd_mod.hip — the single-pass kernel (gqa_fwd_kernel.hpp) with changed
// scores (gqa_score.hpp).
#include "gqa_fwd_kernel.hpp"

namespace gqa {

hipError_t launch_fwd_mod(const FwdParams& p, int dtype, hipStream_t stream, const ScoreMod& mod) {
  FwdModParams m;
  static_cast<FwdParams&>(m) = p;
  m.mod = mod;
  return p.block_table == nullptr ? launch_fwd_pg<0>(m, dtype, stream) : launch_paged_fwd_p(m, dtype, stream);
}

}  // namespace gqa
