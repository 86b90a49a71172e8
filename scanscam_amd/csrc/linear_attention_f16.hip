// Linear attention's kernels for _Float16 activations (fp32 states).
#include "linear_attention_kernels.hpp"

namespace scanscam {
SCANSCAM_DEFINE_ATTEND_LAUNCH(_Float16)
}  // namespace scanscam
