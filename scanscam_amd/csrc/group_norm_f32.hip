// Group norm's kernels for float activations (fp32 arithmetic).
#include "group_norm_kernels.hpp"

namespace scanscam {
SCANSCAM_DEFINE_GROUP_NORM_LAUNCH(float)
}  // namespace scanscam
