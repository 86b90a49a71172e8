// Linear attention's kernels for __bf16 activations (fp32 states).
#include "linear_attention_kernels.hpp"

namespace scanscam {
SCANSCAM_DEFINE_ATTEND_LAUNCH(__bf16)
}  // namespace scanscam
