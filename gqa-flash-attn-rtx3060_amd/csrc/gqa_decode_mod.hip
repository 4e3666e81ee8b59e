// gqa_decode_mod.hip — the decode-shaped first passes (gqa_decode_kernel.hpp)
// with changed scores (gqa_score.hpp); two-launch form only.
#include "gqa_decode_kernel.hpp"

namespace gqa {

hipError_t launch_decode_first_mod(const SplitParams& p, int dtype, hipStream_t stream, const ScoreMod& mod) {
  if (p.counters != nullptr) return hipErrorInvalidValue;
  SplitModParams m;
  static_cast<SplitParams&>(m) = p;
  m.mod = mod;
  return launch_decode_p(m, dtype, stream);
}

}  // namespace gqa
