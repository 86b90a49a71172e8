// Group norm's kernels for _Float16 activations (fp32 arithmetic).
#include "group_norm_kernels.hpp"

namespace scanscam {
SCANSCAM_DEFINE_GROUP_NORM_LAUNCH(_Float16)
}  // namespace scanscam
