// Linear attention's kernels for float activations (fp32 states).
#include "linear_attention_kernels.hpp"

namespace scanscam {
SCANSCAM_DEFINE_ATTEND_LAUNCH(float)
}  // namespace scanscam
