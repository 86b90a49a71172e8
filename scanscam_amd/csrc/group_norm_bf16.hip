// Group norm's kernels for __bf16 activations (fp32 arithmetic).
#include "group_norm_kernels.hpp"

namespace scanscam {
SCANSCAM_DEFINE_GROUP_NORM_LAUNCH(__bf16)
}  // namespace scanscam
