// Norm kernels for __bf16 activations (fp32 arithmetic).
#include "rms_norm_kernels.hpp"

namespace scanscam {
SCANSCAM_DEFINE_NORM_LAUNCH(__bf16)
}  // namespace scanscam
