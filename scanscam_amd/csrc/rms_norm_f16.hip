// Norm kernels for _Float16 activations (fp32 arithmetic).
#include "rms_norm_kernels.hpp"

namespace scanscam {
SCANSCAM_DEFINE_NORM_LAUNCH(_Float16)
}  // namespace scanscam
