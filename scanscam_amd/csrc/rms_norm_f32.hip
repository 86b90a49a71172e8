// Norm kernels for float activations (fp32 arithmetic).
#include "rms_norm_kernels.hpp"

namespace scanscam {
SCANSCAM_DEFINE_NORM_LAUNCH(float)
}  // namespace scanscam
